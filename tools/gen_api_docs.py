"""Writes docs/api/<module>.md: every public name of the package with its signature and the first
paragraph of its docstring (the reference documents one class per page under docs/source/api)."""
import importlib
import inspect
import re
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

MODULES = [
    "evox_amd", "evox_amd.core.random", "evox_amd.core.distributed", "evox_amd.workflows", "evox_amd.parallel",
    "evox_amd.algorithms", "evox_amd.algorithms.so", "evox_amd.algorithms.mo", "evox_amd.algorithms.containers",
    "evox_amd.problems.numerical", "evox_amd.problems.neuroevolution", "evox_amd.problems.evoxbench",
    "evox_amd.operators", "evox_amd.operators.crossover", "evox_amd.operators.mutation", "evox_amd.operators.selection",
    "evox_amd.operators.sampling", "evox_amd.operators.gaussian_process", "evox_amd.monitors", "evox_amd.metrics",
    "evox_amd.utils", "evox_amd.vis_tools.plot", "evox_amd.models", "evox_amd.ops.blas", "evox_amd.ops.sort",
    "evox_amd.ops.gemm", "evox_amd.ops.cma", "evox_amd.ops.nds", "evox_amd.ops.es", "evox_amd.ops.de",
    "evox_amd.ops.variation", "evox_amd.ops.de_adapt", "evox_amd.parallel.p2p", "evox_amd.ops.fitness", "evox_amd.ops.swarm", "evox_amd.ops.moselect", "evox_amd.ops.hv",
    "evox_amd.ops.distance", "evox_amd.ops.linalg_small", "evox_amd.ops.lowrank", "evox_amd.ops.adamw", "evox_amd.utils.optimizers",
    "evox_amd.utils.graph", "evox_amd.utils.profiling",
]


def first_paragraph(obj):
    doc = obj.__doc__ if not inspect.ismodule(obj) else inspect.getdoc(obj)
    if not doc and not inspect.ismodule(obj):
        # undocumented class / function: its module's docstring describes it (one algorithm per file)
        home = sys.modules.get(getattr(obj, "__module__", ""), None)
        doc = inspect.getdoc(home) if home is not None else ""
    doc = inspect.cleandoc(doc or "")
    return doc.split("\n\n")[0].replace("\n", " ").strip()


def signature(obj):
    try:
        # object addresses in default values (<built-in method mean of type object at 0x7f…>) would change on every run
        return re.sub(r" at 0x[0-9a-fA-F]+", "", str(inspect.signature(obj)))
    except (TypeError, ValueError):
        return "(...)"


def public_names(mod):
    names = getattr(mod, "__all__", None)
    if names is None:
        names = [n for n in dir(mod) if not n.startswith("_")]
    out = []
    for n in sorted(names):
        try:
            obj = getattr(mod, n)
        except Exception:
            continue
        if inspect.ismodule(obj):
            continue
        home = getattr(obj, "__module__", "") or ""
        if (inspect.isclass(obj) or inspect.isfunction(obj)) and home.startswith("evox_amd"):
            out.append((n, obj))
    return out


def render(modname):
    mod = importlib.import_module(modname)
    lines = [f"# `{modname}`", "", first_paragraph(mod), ""]
    for name, obj in public_names(mod):
        kind = "class" if inspect.isclass(obj) else "def"
        sig = signature(obj.__init__) if inspect.isclass(obj) and obj.__init__ is not object.__init__ else signature(obj)
        sig = sig.replace("(self, ", "(").replace("(self)", "()")
        lines.append(f"### `{kind} {name}{sig}`")
        lines.append("")
        doc = first_paragraph(obj)
        if doc:
            lines.append(doc)
            lines.append("")
        if inspect.isclass(obj):
            methods = [m for m, f in inspect.getmembers(obj, inspect.isfunction)
                       if not m.startswith("_") and f.__qualname__.startswith(obj.__name__ + ".")]
            if methods:
                lines.append("Methods: " + ", ".join(f"`{m}`" for m in methods))
                lines.append("")
    return "\n".join(lines)


def main():
    out_dir = os.path.join(ROOT, "docs", "api")
    os.makedirs(out_dir, exist_ok=True)
    index = ["# API reference", "", "Generated by `tools/gen_api_docs.py` from the docstrings.", ""]
    for m in MODULES:
        text = render(m)
        fn = m.replace("evox_amd.", "").replace(".", "_") + ".md" if m != "evox_amd" else "evox_amd.md"
        with open(os.path.join(out_dir, fn), "w") as f:
            f.write(text + "\n")
        index.append(f"* [`{m}`]({fn})")
    with open(os.path.join(out_dir, "index.md"), "w") as f:
        f.write("\n".join(index) + "\n")
    print(f"wrote {len(MODULES) + 1} files to {out_dir}")


if __name__ == "__main__":
    main()
