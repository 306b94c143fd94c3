#!/usr/bin/env python3
"""Generates arrowspace-rs_amd/host/rust/src/hip.rs, the `extern "C"` block a maintainer of the reference crate adds
(INTEGRATION.md section 2), from include/arrowspace_hip.h: every export of the header, nothing else.  The image has no
Rust toolchain, so the file is NOT compiled here; tests/test_abi.py checks that it lists exactly the header's exports
and that the committed file is what this script produces.
usage: gen_rust_bindings.py [--check]"""
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HDR = os.path.join(ROOT, "include", "arrowspace_hip.h")
OUT = os.path.join(ROOT, "arrowspace-rs_amd", "host", "rust", "src", "hip.rs")

TYPES = {
    "int": "c_int", "double": "f64", "float": "f32", "uint64_t": "u64", "uint32_t": "u32", "int64_t": "i64", "int32_t": "i32",
    "uint8_t": "u8",
    "void": None,
}
OPAQUE = {"as_ctx": "AsCtx", "as_csr": "AsCsr", "as_index": "AsIndex", "as_graph_params": "AsGraphParams",
          "as_jl": "AsJl", "as_comm": "AsComm", "as_comm_ops": "AsCommOps", "as_clustering": "AsClustering",
          "as_table4": "AsTable4"}


def rust_type(c):
    c = c.strip()
    const = c.startswith("const ")
    base = c[6:] if const else c
    stars = base.count("*")
    base = base.replace("*", "").strip()
    if base == "char":
        t = "c_char"
    elif base == "void":
        t = "c_void"
    elif base in OPAQUE:
        t = OPAQUE[base]
    else:
        t = TYPES[base]
    if stars == 0:
        return t
    out = t
    for level in range(stars):
        inner_const = const and level == 0
        out = ("*const " if inner_const else "*mut ") + out
    return out


def parse():
    src = open(HDR).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    protos = re.findall(r"^((?:const )?[a-z_0-9]+ \*?)\s*(as_\w+)\s*\(([^;{]*?)\);", src, flags=re.M | re.S)
    out = []
    for ret, name, args in protos:
        args = " ".join(args.split())
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                m = re.match(r"(.*?)(\w+)$", a)
                params.append((m.group(2), rust_type(m.group(1))))
        r = ret.strip()
        out.append((name, params, None if r == "void" else rust_type(r)))
    return out


def abi_version():
    return int(re.search(r"#define\s+AS_ABI_VERSION\s+(\d+)", open(HDR).read()).group(1))


def render():
    lines = [
        "// hip.rs -- bindings to include/arrowspace_hip.h (link: -larrowspace_hip).  GENERATED by scripts/gen_rust_bindings.py",
        "// from the header: every export, nothing else.  NOT COMPILED in the build image (no rustc there); the same ABI is",
        "// exercised from C++ (host/arrowspace.hpp, tests/cpp/test_host_mirror.cpp) and from Python (arrowspace_amd/_lib.py).",
        "#![allow(non_camel_case_types, dead_code)]",
        "use std::os::raw::{c_char, c_int, c_void};",
        "",
        "/// include/arrowspace_hip.h: AS_ABI_VERSION.  The ONE place the Rust side reads the expected version from",
        "/// (shim.rs compares as_abi_version() with it; tests/test_abi.py fails on a literal anywhere else).",
        "pub const AS_ABI_VERSION: c_int = %d;" % abi_version(),
        "",
        "#[repr(C)]",
        "#[derive(Clone, Copy, Debug)]",
        "pub struct AsGraphParams {",
        "    // mirrors GraphParams, src/graph.rs:94-102, plus the two CosinePair variant flags of SURVEY.md Appendix A",
        "    pub eps: f64,",
        "    pub k: u64,",
        "    pub topk: u64,",
        "    pub p: f64,",
        "    pub sigma: f64,",
        "    pub has_sigma: i32,",
        "    pub normalise: i32,",
        "    pub sparsity_check: i32,",
        "    pub rectify: i32,",
        "    pub self_in_results: i32,",
        "    pub reserved: i32,",
        "}",
    ]
    protos = parse()
    used = set()
    for _, params, ret in protos:
        for _, t in params:
            used.add(t.split(" ")[-1])
        if ret:
            used.add(ret.split(" ")[-1])
    if "AsCommOps" in used:
        lines += [
            "#[repr(C)]",
            "#[derive(Clone, Copy)]",
            "pub struct AsCommOps {",
            "    // the caller's transport for the sharded build: three primitives over device buffers (see the header)",
            "    pub user: *mut c_void,",
            "    pub all_gather_v: Option<unsafe extern \"C\" fn(*mut c_void, *const c_void, u64, *mut c_void, *const u64, *const u64, *mut c_void) -> c_int>,",
            "    pub all_to_all_v: Option<unsafe extern \"C\" fn(*mut c_void, *const c_void, *const u64, *const u64, *mut c_void, *const u64, *const u64, *mut c_void) -> c_int>,",
            "    pub all_reduce_sum_u64: Option<unsafe extern \"C\" fn(*mut c_void, *mut u64, u64, *mut c_void) -> c_int>,",
            "}",
        ]
    for c, r in OPAQUE.items():
        if r not in ("AsGraphParams", "AsCommOps") and r in used:
            lines += ["#[repr(C)]", "pub struct %s {" % r, "    _private: [u8; 0],", "}"]
    lines += ["", '#[link(name = "arrowspace_hip")]', 'extern "C" {']
    for name, params, ret in protos:
        sig = ", ".join("%s: %s" % (("r#" + n) if n in ("in", "type", "ref", "box") else n, t) for n, t in params)
        lines.append("    pub fn %s(%s)%s;" % (name, sig, (" -> " + ret) if ret else ""))
    lines += ["}", ""]
    return "\n".join(lines), [p[0] for p in protos]


if __name__ == "__main__":
    text, names = render()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == text else 1)
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    open(OUT, "w").write(text)
    print("wrote %s: %d exports" % (OUT, len(names)))
