"""Writes src/cuda_ffi.rs: one `extern "C"` declaration per function of include/flat_attention_b200.h.

    python rust/gen_ffi.py            # rewrites rust/src/cuda_ffi.rs
    python rust/gen_ffi.py --check    # exits 1 if the committed file is stale

The header is the single source of the C ABI; the structs it defines are mirrored by hand in
src/cuda_types.rs (their layout is checked by tests/abi_layout.rs against sizes the library reports).
"""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "include", "flat_attention_b200.h")
OUT = os.path.join(HERE, "src", "cuda_ffi.rs")

SCALARS = {"int32_t": "i32", "uint32_t": "u32", "int64_t": "i64", "uint64_t": "u64", "float": "f32", "double": "f64",
           "char": "c_char", "void": "c_void", "uint16_t": "u16", "uint8_t": "u8", "int": "i32"}
STRUCTS = {"flat_attention_shape": "FlatAttentionShape", "flat_attention_config": "FlatAttentionConfigRaw",
           "flat_rotary_config": "FlatRotaryConfig", "flat_buffer": "FlatBuffer", "flat_forward_layout": "FlatForwardLayout",
           "flat_decode_layout": "FlatDecodeLayout", "flat_backward_layout": "FlatBackwardLayout",
           "flat_varlen_sequence": "FlatVarlenSequence", "flat_paged_kv_telemetry": "FlatPagedKvTelemetry",
           "flat_paged_kv_address": "FlatPagedKvAddress", "flat_numerical_guarantees": "FlatNumericalGuarantees",
           "flat_device_fingerprint": "FlatDeviceFingerprint", "flat_device_capabilities": "FlatDeviceCapabilities",
           "flat_dispatch_telemetry": "FlatDispatchTelemetry", "flat_paged_batch": "FlatPagedBatch",
           "flat_benchmark_manifest": "FlatBenchmarkManifest"}
OPAQUE = {"flat_ctx": "FlatCtx", "flat_paged_kv_table": "FlatPagedKvTable", "flat_paged_kv_cache": "FlatPagedKvCache",
          "flat_resident_kv_cache": "FlatResidentKvCache", "flat_prepared_forward": "FlatPreparedForward",
          "flat_prepared_backward": "FlatPreparedBackward", "flat_splitkv_exchange": "FlatSplitKvExchange"}


def rust_type(c: str) -> str:
    c = c.strip()
    const = False
    stars = c.count("*")
    c = c.replace("*", " ")
    words = [w for w in c.split() if w not in ("struct",)]
    if "const" in words:
        const = True
        words.remove("const")
    base = words[0]
    t = SCALARS.get(base) or STRUCTS.get(base) or OPAQUE.get(base)
    if t is None:
        raise SystemExit("unknown C type in header: %r" % c)
    for i in range(stars):
        t = ("*const " if const and i == stars - 1 or const and stars == 1 else "*mut ") + t
    return t


def functions():
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    text = re.sub(r"^\s*#.*$", "", text, flags=re.M)
    out = []
    for m in re.finditer(r"([A-Za-z_][A-Za-z0-9_ \*]*?)\b(flat_[a-z0-9_]+)\s*\(([^;{}]*?)\)\s*;", text, flags=re.S):
        ret, name, args = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        if ret.startswith("typedef") or "(" in ret:
            continue
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                arr = re.match(r"(.*?)([A-Za-z_][A-Za-z0-9_]*)\[\d*\]$", a)  # `char out[17]` decays to a pointer
                if arr:
                    a = "%s *%s" % (arr.group(1).strip(), arr.group(2))
                pm = re.match(r"(.*?)([A-Za-z_][A-Za-z0-9_]*)$", a)
                params.append((pm.group(2), rust_type(pm.group(1))))
        out.append((name, rust_type(ret) if ret != "void" else None, params))
    return out


def render() -> str:
    lines = ["// Generated by rust/gen_ffi.py from include/flat_attention_b200.h - do not edit by hand.",
             "// One declaration per function of the C ABI of libflat_attention_b200.",
             "#![allow(clippy::too_many_arguments)]", "",
             "use core::ffi::{c_char, c_void};", "", "use crate::cuda_types::*;", "",
             '#[link(name = "flat_attention_b200")]', 'extern "C" {']
    for name, ret, params in functions():
        args = ", ".join("%s: %s" % (("r#" + n) if n in ("type", "in", "ref", "box") else n, t) for n, t in params)
        lines.append("    pub fn %s(%s)%s;" % (name, args, (" -> " + ret) if ret else ""))
    lines += ["}", ""]
    return "\n".join(lines)


if __name__ == "__main__":
    text = render()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == text else 1)
    open(OUT, "w").write(text)
    print("wrote", OUT, "with", len(functions()), "functions")
