"""Generates ``homura_b200/ffi.py`` (ctypes declarations) from ``include/homura_cuda*.h``.

The counterpart of homura's ``tools/gen_rocm_ffi.py``, which runs bindgen over ``csrc/homura_rocm.h`` and
commits the result: here the header is plain enough to read with a small parser, and the committed
``ffi.py`` is compared against a fresh generation with ``--check`` (the test suite does that), so header and
binding cannot drift apart. A Rust integration would run bindgen with the allow-list ``hmc_.*|HMC_.*`` instead.

    python -m homura_b200.gen_cuda_ffi           # rewrite ffi.py
    python -m homura_b200.gen_cuda_ffi --check   # exit 1 if ffi.py is stale
"""
from __future__ import annotations

import re
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
HEADERS = [ROOT / "include" / "homura_cuda.h", ROOT / "include" / "homura_cuda_alloc.h",
           ROOT / "include" / "homura_cuda_shard.h", ROOT / "include" / "homura_cuda_layers.h"]
OUT = Path(__file__).resolve().parent / "ffi.py"

CTYPES = {
    "void": None,
    "char": "c_char",
    "int32_t": "c_int32",
    "uint32_t": "c_uint32",
    "int64_t": "c_int64",
    "uint64_t": "c_uint64",
    "uint8_t": "c_uint8",
    "float": "c_float",
    "double": "c_double",
    "hmc_status": "c_int32",
}


def strip_comments(text: str) -> str:
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def ctype(decl: str, structs: set[str], handles: set[str]) -> str:
    """The ctypes expression of a C type such as ``const hmc_tensor_desc *`` or ``void **``."""
    decl = decl.replace("const", " ").replace("struct", " ").strip()
    stars = decl.count("*")
    base = decl.replace("*", " ").split()[0]
    if base in handles:
        expr, stars = "c_void_p", stars
    elif base in structs:
        expr = base
    elif base == "void":
        if stars == 0:
            return "None"
        expr, stars = "c_void_p", stars - 1
    elif base == "char" and stars >= 1:
        expr, stars = "c_char_p", stars - 1
    else:
        expr = CTYPES[base]
    for _ in range(stars):
        expr = f"POINTER({expr})"
    return expr


def parse(text: str):
    text = strip_comments(text)
    defines = re.findall(r"^#define\s+(HMC_\w+)\s+(-?\d+)\s*$", text, flags=re.M)
    handles = set(re.findall(r"typedef\s+struct\s+\w+\s*\*\s*(\w+)\s*;", text))
    structs = []
    for body, name in re.findall(r"typedef\s+struct\s+\w+\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
        fields = []
        for line in body.split(";"):
            line = " ".join(line.split())
            if not line:
                continue
            fp = re.match(r"(.+?)\(\s*\*\s*(\w+)\s*\)\s*\((.*)\)$", line)
            if fp:
                # a function pointer field: ("fn:<ret>|<arg>,<arg>", name, None)
                args = [re.match(r"(.+?)(\w+)$", a.strip()).group(1).strip() for a in fp.group(3).split(",")]
                fields.append(("fn:" + fp.group(1).strip() + "|" + ",".join(args), fp.group(2), None))
                continue
            m = re.match(r"(.+?)\s*(\**)\s*(\w+)\s*(\[(\w+)\])?$", line)
            typ, stars, fname, _, dim = m.groups()
            fields.append((typ + stars, fname, dim))
        structs.append((name, fields))
    body = re.sub(r"typedef\s+struct\s+\w+\s*\{.*?\}\s*\w+\s*;", "", text, flags=re.S)
    body = re.sub(r"typedef[^;]*;", "", body)
    body = re.sub(r"^#.*$", "", body, flags=re.M)
    body = body.replace('extern "C" {', "").replace("}", "")
    functions = []
    for stmt in body.split(";"):
        stmt = " ".join(stmt.split())
        m = re.match(r"(.+?)\s*(\**)\s*(hmc_\w+)\s*\((.*)\)$", stmt)
        if not m:
            continue
        ret, rstars, name, args = m.groups()
        params = []
        if args.strip() != "void":
            for a in args.split(","):
                a = a.strip()
                pm = re.match(r"(.+?)(\w+)$", a)
                params.append((pm.group(1).strip(), pm.group(2)))
        functions.append((ret + rstars, name, params))
    return defines, handles, structs, functions


def generate() -> str:
    defines, handles, structs, functions = [], set(), [], []
    for h in HEADERS:
        if not h.exists():
            continue
        d, hd, s, f = parse(h.read_text())
        defines += d
        handles |= hd
        structs += s
        functions += f
    names = {n for n, _ in structs}
    consts = dict(defines)
    out = [
        '"""ctypes declarations of the C ABI in include/homura_cuda*.h.',
        "",
        "GENERATED by homura_b200/gen_cuda_ffi.py; do not edit (the tests run the generator with --check).",
        '"""',
        "from ctypes import (CFUNCTYPE, POINTER, Structure, c_char, c_char_p, c_double, c_float, c_int32, c_int64, c_uint8,",
        "                    c_uint32, c_uint64, c_void_p)",
        "",
    ]
    for k, v in defines:
        out.append(f"{k} = {v}")
    out.append("")
    for name, fields in structs:
        out.append("")
        out.append(f"class {name}(Structure):")
        out.append("    _fields_ = [")
        for typ, fname, dim in fields:
            if typ.startswith("fn:"):
                ret, args = typ[3:].split("|")
                parts = [ctype(ret, names, handles)] + [ctype(a, names, handles) for a in args.split(",")]
                out.append(f'        ("{fname}", CFUNCTYPE({", ".join(parts)})),')
                continue
            expr = ctype(typ, names, handles)
            if dim is not None:
                n = consts.get(dim, dim)
                expr = f"{expr} * {n}"
            out.append(f'        ("{fname}", {expr}),')
        out.append("    ]")
        out.append("")
    out.append("")
    out.append("# name -> (restype, [(argtype, argname), ...])")
    out.append("FUNCTIONS = {")
    for ret, name, params in functions:
        args = ", ".join(f'({ctype(t, names, handles)}, "{n}")' for t, n in params)
        out.append(f'    "{name}": ({ctype(ret, names, handles)}, [{args}]),')
    out.append("}")
    out.append("")
    out.append("")
    out.append("def bind(lib, only=None):")
    out.append('    """Sets restype/argtypes on every declared function `lib` exports; returns the names bound."""')
    out.append("    bound = []")
    out.append("    for name, (res, params) in FUNCTIONS.items():")
    out.append("        if only is not None and name not in only:")
    out.append("            continue")
    out.append("        fn = getattr(lib, name, None)")
    out.append("        if fn is None:")
    out.append("            continue")
    out.append("        fn.restype = res")
    out.append("        fn.argtypes = [t for t, _ in params]")
    out.append("        bound.append(name)")
    out.append("    return bound")
    out.append("")
    return "\n".join(out)


def main() -> int:
    text = generate()
    if "--check" in sys.argv:
        if not OUT.exists() or OUT.read_text() != text:
            print("homura_b200/ffi.py is stale: run python -m homura_b200.gen_cuda_ffi", file=sys.stderr)
            return 1
        return 0
    OUT.write_text(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
