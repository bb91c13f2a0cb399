"""Writes the reference of the Python layer from the code itself: for every public module its classes (with their public
methods) and functions, each with its signature and the first paragraph of its docstring.

    python -m rocm_systems_b200.utils.apidoc > docs/python_api.md
    python -m rocm_systems_b200.utils.apidoc --c > docs/c_api.md      # the C and device API, from the public headers
"""
from __future__ import annotations

import importlib
import inspect
import sys
from typing import List

MODULES = [
    "rocm_systems_b200.comm", "rocm_systems_b200.shmem",
    "rocm_systems_b200.parallel.dist", "rocm_systems_b200.parallel.fsdp", "rocm_systems_b200.parallel.tp", "rocm_systems_b200.parallel.ep",
    "rocm_systems_b200.parallel.pp", "rocm_systems_b200.parallel.cp",
    "rocm_systems_b200.models.llama", "rocm_systems_b200.ops.train_ops", "rocm_systems_b200.ops.attention", "rocm_systems_b200.ops.fp8",
    "rocm_systems_b200.utils.checkpoint", "rocm_systems_b200.utils.elastic", "rocm_systems_b200.utils.markers", "rocm_systems_b200.utils.profiler",
    "rocm_systems_b200.utils.causal", "rocm_systems_b200.utils.affinity", "rocm_systems_b200.utils.hang_dump",
    "rocm_systems_b200.tools.smi", "rocm_systems_b200.tools.telemetry", "rocm_systems_b200.tools.tracedb", "rocm_systems_b200.tools.counters",
    "rocm_systems_b200.tools.causal", "rocm_systems_b200.tools.pytrace", "rocm_systems_b200.tools.instrument", "rocm_systems_b200.tools.sysmon",
]


def first_paragraph(obj) -> str:
    doc = inspect.getdoc(obj) or ""
    para = doc.split("\n\n", 1)[0].replace("\n", " ").strip()
    return para


def signature(obj) -> str:
    try:
        return str(inspect.signature(obj)).replace("'", "").replace('"', "")   # annotations are kept as text: drop their quotes
    except (TypeError, ValueError):
        return "(...)"


def describe(module_name: str) -> List[str]:
    mod = importlib.import_module(module_name)
    out = [f"## `{module_name}`", "", first_paragraph(mod), ""]
    members = [(n, o) for n, o in vars(mod).items() if not n.startswith("_") and getattr(o, "__module__", None) == module_name]
    for name, obj in members:
        if inspect.isclass(obj):
            out.append(f"### class `{name}{signature(obj)}`")
            para = first_paragraph(obj)
            if para:
                out += ["", para]
            out.append("")
            for mname, meth in vars(obj).items():
                if mname.startswith("_") or not (inspect.isfunction(meth) or isinstance(meth, (staticmethod, classmethod, property))):
                    continue
                target = meth.fget if isinstance(meth, property) else (meth.__func__ if isinstance(meth, (staticmethod, classmethod)) else meth)
                kind = "property " if isinstance(meth, property) else ""
                line = f"- {kind}`{mname}{'' if isinstance(meth, property) else signature(target)}`"
                para = first_paragraph(target)
                out.append(line + (f": {para}" if para else ""))
            out.append("")
    for name, obj in members:
        if inspect.isfunction(obj):
            para = first_paragraph(obj)
            out.append(f"- `{name}{signature(obj)}`" + (f": {para}" if para else ""))
    out.append("")
    return out


def c_reference() -> List[str]:
    """The C and device API from the public headers: every function with its prototype and the comment that stands right
    above it (``B200COLL_DECL`` entries of nccl.h, plain prototypes, and the ``__device__`` functions of shmem_device.cuh)."""
    import re
    from pathlib import Path

    inc = Path(__file__).resolve().parents[1] / "csrc" / "include" / "b200coll"
    out = ["# C and device API reference", "",
           "Generated by `python -m rocm_systems_b200.utils.apidoc --c` from the public headers under `csrc/include/b200coll/`: every function "
           "with its prototype and the comment right above it. `api.md` explains how the parts belong together.", ""]
    decl = re.compile(r"B200COLL_DECL\(\s*([^,]+?)\s*,\s*(\w+)\s*,\s*(.*?)\)\s*$", re.S)
    proto = re.compile(r"^(?!typedef|#|static|return|extern \"C\")([A-Za-z_][\w\s\*]*?[\s\*])(\w+)\s*\(([^;{}]*)\)\s*;", re.S)
    dev = re.compile(r"__device__\s+(?:__forceinline__\s+|inline\s+)*([\w:<>\*&\s]+?[\s\*&])(\w+)\s*\(([^)]*)\)\s*(?:const\s*)?\{", re.S)

    def squash(t: str) -> str:
        return re.sub(r"\s+", " ", t).strip()

    def comment_above(text: str, pos: int) -> str:
        head = text[:pos].rstrip()
        if head.endswith("*/"):
            start = head.rfind("/*")
            body = head[start + 2:-2]
            body = re.sub(r"^\s*\*+\s?", "", body, flags=re.M)
            return squash(body)
        lines = []
        for line in reversed(head.splitlines()):
            if line.strip().startswith("//"):
                lines.append(line.strip()[2:].strip())
            else:
                break
        return squash(" ".join(reversed(lines)))

    for h in sorted(inc.iterdir()):
        if h.suffix not in (".h", ".cuh"):
            continue
        text = h.read_text()
        found = []
        if h.suffix == ".cuh":
            for m in dev.finditer(text):
                name = m.group(2)
                if not name.startswith("_") and not name.endswith("_"):
                    found.append((m.start(), f"{squash(m.group(1))} {name}({squash(m.group(3))})", comment_above(text, m.start())))
        else:
            for m in re.finditer(r"B200COLL_DECL\((?:[^()]|\([^()]*\))*\)", text):
                d = decl.match(m.group(0))
                if d:
                    found.append((m.start(), f"{squash(d.group(1))} {d.group(2)}({squash(d.group(3))})", comment_above(text, m.start())))
            for chunk in re.finditer(r"(?m)^[A-Za-z_][^;{}#]*\([^;{}]*\)\s*;", text):
                m = proto.match(chunk.group(0))
                if m and not m.group(2).startswith("_") and "(" not in m.group(1):
                    found.append((chunk.start(), f"{squash(m.group(1))} {m.group(2)}({squash(m.group(3))})", comment_above(text, chunk.start())))
        if not found:
            continue
        out += [f"## `b200coll/{h.name}`", ""]
        seen = set()
        for _, sig, note in sorted(found):
            note = re.sub(r"-{4,}.*?-{4,}", "", note).strip()      # section dividers are not descriptions
            if sig in seen or sig.startswith("ret name("):           # the declaration macro's own definition
                continue
            seen.add(sig)
            out.append(f"- `{sig}`" + (f": {note}" if note else ""))
        out.append("")
    return out


def main(argv=None) -> int:
    argv = list(sys.argv[1:] if argv is None else argv)
    if "--c" in argv:
        sys.stdout.write("\n".join(c_reference()) + "\n")
        return 0
    lines = ["# Python reference", "",
             "Generated by `python -m rocm_systems_b200.utils.apidoc` from the signatures and docstrings of the code; the guide (`guide.md`) shows "
             "how the pieces are used together.", ""]
    for m in MODULES:
        try:
            lines += describe(m)
        except Exception as e:  # noqa: BLE001  a module that cannot be imported here is named, not fatal
            lines += [f"## `{m}`", "", f"(not importable here: {type(e).__name__}: {e})", ""]
    sys.stdout.write("\n".join(lines) + "\n")
    return 0


if __name__ == "__main__":
    sys.exit(main())
