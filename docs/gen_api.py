"""Regenerates docs/api.md: the public names of every user-facing module with their signatures and the first line of
their docstrings.

    python docs/gen_api.py
"""
import importlib
import inspect
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

MODULES = [
    "genesis_b200", "genesis_b200.nn", "genesis_b200.nn.functional", "genesis_b200.nn.utils", "genesis_b200.nn.parallel", "genesis_b200.nn.paged",
    "genesis_b200.optim", "genesis_b200.optim.lr_scheduler", "genesis_b200.amp", "genesis_b200.cuda",
    "genesis_b200.distributed", "genesis_b200.distributed.symm", "genesis_b200.distributed.watchdog",
    "genesis_b200.parallel.ep", "genesis_b200.models.transformers", "genesis_b200.serialization",
    "genesis_b200.utils.data", "genesis_b200.utils.profile", "genesis_b200.utils.metrics", "genesis_b200.backends",
    "genesis_b200.ops.dispatch",
]


def first_line(obj):
    # the object's own docstring only: inherited ones (Function subclasses, enums) would repeat their base's line
    d = (vars(obj).get("__doc__") if inspect.isclass(obj) else getattr(obj, "__doc__", None)) or ""
    return d.strip().split("\n")[0] if d.strip() else ""


def sig(obj):
    try:
        return str(inspect.signature(obj))
    except (TypeError, ValueError):
        return "(...)"


def main():
    out = ["# API index", "",
           "Generated by `python docs/gen_api.py` from the docstrings; `import genesis` resolves to the same modules.", ""]
    for name in MODULES:
        m = importlib.import_module(name)
        out.append(f"## `{name.replace('genesis_b200', 'genesis')}`")
        doc = first_line(m)
        if doc:
            out.append(doc)
        out.append("")
        rows = []
        for n in sorted(getattr(m, "__all__", dir(m))):
            if n.startswith("_"):
                continue
            o = getattr(m, n)
            if inspect.ismodule(o):
                continue
            home = getattr(o, "__module__", "") or ""
            if not home.startswith("genesis_b200"):
                continue
            if inspect.isclass(o):
                rows.append(f"* class `{n}{sig(o)}` — {first_line(o)}".rstrip(" —"))
            elif callable(o):
                rows.append(f"* `{n}{sig(o)}` — {first_line(o)}".rstrip(" —"))
        out.extend(rows or ["(re-exports only)"])
        out.append("")
    with open(os.path.join(ROOT, "docs", "api.md"), "w", encoding="utf-8") as f:
        f.write("\n".join(out))
    print(f"docs/api.md: {len(out)} lines")


if __name__ == "__main__":
    main()
