#!/usr/bin/env python
"""Writes src/lib.rs of the mechta-kv-sys crate from include/mechta_kv.h: one `extern "C"` declaration per entry
point of the C ABI, the `#[repr(C)]` structs, the status and format constants.

    python rust/mechta-kv-sys/gen_bindings.py          # rewrites rust/mechta-kv-sys/src/lib.rs
    python rust/mechta-kv-sys/gen_bindings.py --check  # exits 1 if the file on disk differs from what would be written

The header is the single source of truth; tests/test_abi_cpu.py runs the check and also compares names and argument
counts independently of this script. No Rust toolchain is needed to generate; none was available to compile the crate
where it was written, and the file says so.
"""
from __future__ import annotations

import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "mechta_kv.h")
OUT = os.path.join(HERE, "src", "lib.rs")

SCALARS = {"int": "c_int", "uint32_t": "u32", "int32_t": "i32", "uint64_t": "u64", "int64_t": "i64", "size_t": "usize", "float": "f32",
           "double": "f64", "char": "c_char", "void": "c_void", "mkv_status": "mkv_status", "mkv_fmt": "mkv_fmt"}
OPAQUE = ["mkv_ctx", "mkv_cache", "mkv_exchange", "mkv_rope", "mkv_pool"]
STRUCTS = ["mkv_verify_item", "mkv_step_in", "mkv_rope_desc", "mkv_rope_rows", "mkv_pool_desc", "mkv_seq_rows", "mkv_pool_rows",
           "mkv_pool_attn"]


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def rust_type(c: str) -> str:
    """C type (without the parameter name) -> Rust type."""
    c = " ".join(c.replace("*", " * ").split())
    toks = c.split()
    const = False
    base = None
    ptrs = []  # one entry per '*': is the pointee const?
    for t in toks:
        if t == "const":
            const = True
        elif t == "*":
            ptrs.append(const)
            const = False
        else:
            base = t
    ty = SCALARS.get(base, base)
    assert ty is not None and (base in SCALARS or base in OPAQUE or base in STRUCTS), c
    for pointee_const in ptrs:
        ty = ("*const " if pointee_const else "*mut ") + ty
    return ty


def split_param(p: str):
    p = " ".join(p.split())
    m = re.match(r"^(.*?)(\w+)\s*(\[\d+\])?$", p)
    ctype, name, arr = m.group(1).strip(), m.group(2), m.group(3)
    if arr:  # `const uint32_t u[8]` decays to a pointer
        ctype += " *"
    return ctype, name


def functions(text: str):
    out = []
    for m in re.finditer(r"([\w\s\*]+?)\b(mkv_\w+)\s*\(([^;{}]*?)\)\s*;", text):
        ret, name, args = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
        params = [] if args == "void" else [split_param(a) for a in args.split(",")]
        out.append((ret, name, params))
    return out


def structs(text: str):
    out = {}
    for m in re.finditer(r"typedef\s+struct\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
        fields = []
        for decl in m.group(1).split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            head, *more = [x.strip() for x in decl.split(",")]
            ctype, name = split_param(head)
            fields.append((ctype, name))
            for extra in more:  # `uint32_t first_pos, pos, ntok;`
                fields.append((ctype, extra))
        out[m.group(2)] = fields
    return out


def enums(text: str):
    vals = []
    for m in re.finditer(r"\b(MKV_[A-Z0-9_]+)\s*=\s*(\d+)", text):
        vals.append((m.group(1), int(m.group(2))))
    return vals


def render() -> str:
    text = strip_comments(open(HEADER).read())
    fns, sts, consts = functions(text), structs(text), enums(text)
    L = []
    L.append("//! Raw bindings of libmechta_kv (include/mechta_kv.h), the C ABI of the B200 KV-cache / attention path.")
    L.append("//!")
    L.append("//! GENERATED by gen_bindings.py from the header; do not edit by hand. NOT COMPILED where it was written (no Rust")
    L.append("//! toolchain there): names, argument counts and types are checked textually against the header by the test suite.")
    L.append("//! This crate is the one `unsafe` surface of the path, as engine/crates/shader is in the reference; the safe")
    L.append("//! wrapper is the `mechta-kv` crate beside it. Link with `-lmechta_kv` (see build.rs).")
    L.append("#![allow(non_camel_case_types)]")
    L.append("")
    L.append("use core::ffi::{c_char, c_int, c_void};")
    L.append("")
    L.append("pub type mkv_status = c_int;")
    L.append("pub type mkv_fmt = c_int;")
    for name, val in consts:
        ty = "mkv_status" if name.startswith("MKV_OK") or name.startswith("MKV_ERR") else ("mkv_fmt" if name in ("MKV_F16", "MKV_F32") else "c_int")
        L.append(f"pub const {name}: {ty} = {val};")
    L.append("")
    for o in OPAQUE:
        L.append("#[repr(C)]")
        L.append(f"pub struct {o} {{")
        L.append("    _private: [u8; 0],")
        L.append("}")
    L.append("")
    for sname in STRUCTS:
        L.append("#[repr(C)]")
        L.append("#[derive(Clone, Copy)]")
        L.append(f"pub struct {sname} {{")
        for ctype, fname in sts[sname]:
            L.append(f"    pub {fname}: {rust_type(ctype)},")
        L.append("}")
        L.append("")
    L.append('extern "C" {')
    for ret, name, params in fns:
        args = ", ".join(f"{'r#in' if n == 'in' else n}: {rust_type(t)}" for t, n in params)
        r = "" if ret == "void" else f" -> {rust_type(ret)}"
        L.append(f"    pub fn {name}({args}){r};")
    L.append("}")
    L.append("")
    return "\n".join(L)


def main() -> int:
    text = render()
    if "--check" in sys.argv:
        same = os.path.exists(OUT) and open(OUT).read() == text
        if not same:
            print("rust/mechta-kv-sys/src/lib.rs is out of date: run gen_bindings.py", file=sys.stderr)
        return 0 if same else 1
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    open(OUT, "w").write(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
