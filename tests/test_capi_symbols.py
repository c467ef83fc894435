"""CPU: the C-ABI shared library loads, exports EVERY function include/arrow_gpu.h declares (and the ctypes table
matches), and fails loudly without a GPU — no compute calls here."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "arrow_gpu.h")


def declared_functions():
    src = open(HEADER).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(agpu_[a-z0-9_]+)\s*\(", src)))


def test_header_declares_the_documented_surface():
    fns = declared_functions()
    assert len(fns) >= 55
    for must in ("agpu_device_create", "agpu_pipeline_create", "agpu_binary", "agpu_scalar", "agpu_unary", "agpu_cast",
                 "agpu_compare", "agpu_compare_validity", "agpu_bitmap_binary", "agpu_bitmap_popcount", "agpu_reduce",
                 "agpu_take", "agpu_put", "agpu_merge", "agpu_broadcast", "agpu_launch_by_name"):
        assert must in fns


def test_library_exports_every_declared_symbol():
    from arrow_gpu_amd import _capi as capi

    lib = capi.lib()
    missing = [f for f in declared_functions() if not hasattr(lib, f)]
    assert not missing, f"declared in include/arrow_gpu.h but not exported: {missing}"


def test_ctypes_table_covers_header():
    from arrow_gpu_amd import _capi as capi

    declared = set(declared_functions())
    bound = set(capi.SIGNATURES)
    assert declared - bound == set(), f"unbound: {sorted(declared - bound)}"
    assert bound - declared == set(), f"bound but undeclared: {sorted(bound - declared)}"


def test_misc_queries_work_without_gpu():
    from arrow_gpu_amd import _capi as capi

    lib = capi.lib()
    assert lib.agpu_abi_version() == 2
    assert b"gfx950" in lib.agpu_build_info()
    assert lib.agpu_dtype_size(capi.F32) == 4 and lib.agpu_dtype_size(capi.I16) == 2 and lib.agpu_dtype_size(capi.BOOL) == 0
    assert lib.agpu_bitmap_bytes(0) == 0 and lib.agpu_bitmap_bytes(1) == 8 and lib.agpu_bitmap_bytes(65) == 16
    v = C.c_int64(-1)
    assert lib.agpu_get_tuning(b"stream_grid", C.byref(v)) == 0
    assert lib.agpu_set_tuning(b"no_such_key", 1) == capi.ERR_ARG


def test_the_tuning_keys_are_the_seven_the_header_lists():
    """the public tuning surface was 17 keys, nine of which never beat their default.  The header's list, the library's
    table and the set the ABI fuzz draws (tests/test_gpu_fuzz_abi.py TUNING_KEYS) are the same seven; the removed ones are argument errors."""
    import re

    from arrow_gpu_amd import _capi as capi

    lib = capi.lib()
    header = open(os.path.join(ROOT, "include", "arrow_gpu.h"), encoding="utf-8").read()
    doc = header[header.index("/* Launch tuning"):header.index("agpu_status agpu_set_tuning")]
    listed = re.findall(r'^ \*   "([a-z0-9_]+)"', doc, flags=re.M)
    assert len(listed) == 7 and len(set(listed)) == 7, listed
    v = C.c_int64(-1)
    for key in listed:
        assert lib.agpu_get_tuning(key.encode(), C.byref(v)) == 0 and v.value == 0, key
    for gone in ("stream_bpc", "stream_unroll", "stream_nt", "reduce_grid", "gather_region_bits", "gather_offsets", "h2d_threads",
                 "heavy_tiles", "cast_tiles", "table_tiles", "tile_auto"):
        assert lib.agpu_get_tuning(gone.encode(), C.byref(v)) == capi.ERR_ARG, gone
    fuzz = open(os.path.join(ROOT, "tests", "test_gpu_fuzz_abi.py"), encoding="utf-8").read()
    drawn = re.search(r"^TUNING_KEYS = \(([^)]*)\)", fuzz, flags=re.M).group(1)
    assert sorted(re.findall(r'"([a-z0-9_]+)"', drawn)) == sorted(listed)
    for key in listed:  # … and every one of them is SET inside the fuzz loop
        assert f'set_tuning("{key}"' in fuzz, key


def test_no_cpu_fallback():
    """Without a device the product raises; it never computes on the host."""
    import torch

    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present")
    import arrow_gpu_amd as ag

    with pytest.raises(ag.ArrowErrorGPU) as ei:
        ag.GpuDevice(0)
    assert ei.value.status == 5  # AGPU_ERR_NO_DEVICE


def test_the_product_library_carries_no_test_hook():
    """comm.hip's stall hook (an RCCL bootstrap that does not come up, reproducibly) is compiled into the TEST build only
    (libarrow_gpu_hip_hooks.so, -DAGPU_TEST_HOOKS; tests/test_gpu_comm.py loads it through AGPU_LIB)."""
    import mmap

    def mentions_hook(path):  # (mapped, not read: a 7 MB bytes object freed here would raise glibc's mmap threshold for the tests that follow)
        with open(path, "rb") as f, mmap.mmap(f.fileno(), 0, access=mmap.ACCESS_READ) as m:
            return m.find(b"AGPU_COMM_TEST_STALL_INIT_MS") >= 0

    lib_dir = os.path.join(ROOT, "arrow_gpu_amd", "lib")
    assert not mentions_hook(os.path.join(lib_dir, "libarrow_gpu_hip.so"))
    hooks = os.path.join(lib_dir, "libarrow_gpu_hip_hooks.so")
    assert os.path.exists(hooks), "build() makes the test build too (csrc/Makefile `hooks`)"
    assert mentions_hook(hooks)


def test_product_never_imports_oracle():
    pkg = os.path.join(ROOT, "arrow_gpu_amd")
    for dp, _, fns in os.walk(pkg):
        for fn in fns:
            if fn.endswith((".py", ".hip", ".hpp", ".h", ".inc")):
                text = open(os.path.join(dp, fn)).read()
                assert not re.search(r"^\s*(import|from)\s+oracle\b", text, flags=re.M), f"{fn} imports the oracle"
                assert "liboracle" not in text and "agpu_oracle" not in text.replace("oracle/agpu_oracle.c", ""), fn


# ---------------------------------------------------------------- the Rust side (bindings/rust): generated, and tied to the header
# There is no rustc in the build image, so the binding cannot be compiled here.  What can be checked mechanically is: the committed
# files ARE the generator's output for the current header; every export is declared in ffi.rs with the same arity and the same
# argument / return widths (parsed here INDEPENDENTLY of the generator); the #[repr(C)] structs have the header's fields in the
# header's order; and the two modules carrying the reference's method signatures only call ffi functions that exist, with the right
# number of arguments.  [ref: crates/array/src/gpu_utils/gpu_device.rs:171-509, compute_pipeline.rs:24-299]
RUST_DIR = os.path.join(ROOT, "bindings", "rust")
_C_WIDTH = {"int32_t": "i4", "uint32_t": "i4", "int": "i4", "int64_t": "i8", "uint64_t": "i8", "size_t": "isize", "float": "f4", "double": "f8",
            "uint8_t": "i1", "char": "i1", "void": "void"}
_RUST_WIDTH = {"i32": "i4", "u32": "i4", "c_int": "i4", "i64": "i8", "u64": "i8", "usize": "isize", "f32": "f4", "f64": "f8", "u8": "i1", "c_char": "i1"}


def _split_args(text):
    """top-level commas only"""
    out, depth, cur = [], 0, ""
    for ch in text:
        if ch in "(<[":
            depth += 1
        elif ch in ")>]":
            depth -= 1
        if ch == "," and depth == 0:
            out.append(cur.strip())
            cur = ""
        else:
            cur += ch
    if cur.strip():
        out.append(cur.strip())
    return out


def _header_signatures():
    src = re.sub(r"/\*.*?\*/", " ", open(HEADER).read(), flags=re.S)
    enums = set(re.findall(r"typedef\s+enum\s*\{[^}]*\}\s*(\w+)\s*;", src)) | {"agpu_status"}
    sigs = {}
    for m in re.finditer(r"\n\s*((?:const\s+)?\w+[\s\*]+?)\b(agpu_\w+)\s*\(([^;{}]*?)\)\s*;", src, flags=re.S):
        def width(ctype):
            ctype = ctype.strip()
            if "*" in ctype:
                return "ptr"
            base = ctype.replace("const", "").replace("struct", "").split()[0]
            return "i4" if base in enums else _C_WIDTH[base]

        args = [] if m.group(3).strip() in ("", "void") else [width(re.sub(r"\b\w+$", "", a.strip())) for a in _split_args(" ".join(m.group(3).split()))]
        sigs[m.group(2)] = (width(m.group(1)), args)
    return sigs


def _rust_signatures():
    text = open(os.path.join(RUST_DIR, "ffi.rs")).read()
    aliases = set(re.findall(r"pub type (\w+) = i32;", text))
    sigs = {}
    for m in re.finditer(r"pub fn (agpu_\w+)\((.*?)\)(?: -> ([^;]+))?;", text):
        def width(rt):
            rt = rt.strip()
            if rt.startswith("*"):
                return "ptr"
            return "i4" if rt in aliases else _RUST_WIDTH[rt]

        args = [width(a.split(":", 1)[1]) for a in _split_args(m.group(2))]
        sigs[m.group(1)] = (width(m.group(3)) if m.group(3) else "void", args)
    return sigs


def test_rust_bindings_are_the_generators_output_for_this_header():
    import subprocess
    import sys

    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "gen_rust_ffi.py"), "--check"], capture_output=True, text=True)
    assert r.returncode == 0, "bindings/rust is stale: run `python tools/gen_rust_ffi.py`\n" + r.stdout + r.stderr


def test_rust_ffi_declares_every_export_with_the_headers_arity_and_widths():
    hs, rs = _header_signatures(), _rust_signatures()
    assert set(hs) == set(declared_functions())          # the independent parse sees every export
    assert set(rs) == set(hs), (sorted(set(hs) - set(rs)), sorted(set(rs) - set(hs)))
    bad = {n: (hs[n], rs[n]) for n in hs if hs[n] != rs[n]}
    assert not bad, bad
    assert len(hs) >= 129


def test_rust_structs_mirror_the_headers_fields_in_order():
    src = re.sub(r"/\*.*?\*/", " ", open(HEADER).read(), flags=re.S)
    rust = open(os.path.join(RUST_DIR, "ffi.rs")).read()
    checked = 0
    for m in re.finditer(r"(?:typedef\s+struct\s*\w*|struct\s+(\w+))\s*\{(.*?)\}\s*(\w*)\s*;", src, flags=re.S):
        name = m.group(3) or m.group(1)
        names = []
        for decl in m.group(2).split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            fp = re.match(r".*\(\s*\*\s*(\w+)\s*\)\s*\(", decl)
            if fp:
                names.append(fp.group(1))
            else:
                first = True
                for piece in decl.split(","):
                    nm = re.sub(r"\[\d+\]$", "", piece.strip()).split()[-1].lstrip("*") if not first else re.sub(r"\[\d+\]$", "", piece.strip().split()[-1]).lstrip("*")
                    names.append(nm)
                    first = False
        rm = re.search(r"pub struct %s \{(.*?)\n\}" % re.escape(name), rust, flags=re.S)
        assert rm, f"struct {name} missing from ffi.rs"
        rnames = re.findall(r"pub (\w+):", rm.group(1))
        assert rnames == names, (name, names, rnames)
        assert "#[repr(C)]\npub struct %s {" % name in rust
        checked += 1
    assert checked >= 7
    for opaque in ("agpu_device", "agpu_pipeline", "agpu_event", "agpu_graph", "agpu_comm", "agpu_ipc_reader", "agpu_ipc_writer"):
        assert "#[repr(C)] pub struct %s { _private: [u8; 0] }" % opaque in rust
    for const in ("AGPU_OK", "AGPU_ERR_NO_DEVICE", "AGPU_F32", "AGPU_OP_POW", "AGPU_UN_SINH", "AGPU_CMP_EQ", "AGPU_RED_MAX", "AGPU_COMM_ID_BYTES"):
        assert re.search(r"pub const %s: \w+ = \d+;" % const, rust), const


# the Rust reference, "Keywords": strict ones, those of later editions, reserved ones
_RUST_KEYWORDS = set("""as break const continue crate else enum extern false fn for if impl in let loop match mod move mut pub ref return self Self static
struct super trait true type unsafe use where while async await dyn abstract become box do final macro override priv typeof unsized virtual yield try
gen""".split())


def test_rust_ffi_names_no_keyword():
    """a keyword in the place of a name ends the parse of the whole file: fields, arguments, functions, types and constants"""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(RUST_DIR, "ffi.rs")).read())
    names = []
    for body in re.findall(r"pub struct \w+ \{(.*?)\}", text, flags=re.S):
        names += re.findall(r"(?:^|[,{]|\n)\s*(?:pub\s+)?([\w#]+)\s*:", body)
    for args in re.findall(r"pub fn \w+\((.*?)\)(?: ->|;)", text):
        names += [a.split(":", 1)[0].strip() for a in _split_args(args)]
    names += re.findall(r"pub (?:fn|type|const|struct) ([\w#]+)", text)
    assert len(names) > 500 and "r#in" in names and "row_type" in names
    assert not [n for n in names if n in _RUST_KEYWORDS], sorted(set(names) & _RUST_KEYWORDS)
    raw = {n[2:] for n in names if n.startswith("r#")}
    assert raw <= _RUST_KEYWORDS - {"crate", "self", "Self", "super"}  # those have no raw form


def test_rust_host_modules_call_only_existing_ffi_functions_with_the_right_arity():
    rs = _rust_signatures()
    seen = set()
    for fn in ("gpu_device.rs", "compute_pipeline.rs", "mod.rs"):
        text = open(os.path.join(RUST_DIR, fn)).read()
        for m in re.finditer(r"ffi::(agpu_\w+)\(", text):
            name = m.group(1)
            assert name in rs, f"{fn} calls ffi::{name}, which the header does not declare"
            depth, i = 1, m.end()
            while depth:
                depth += text[i] in "([{"
                depth -= text[i] in ")]}"
                i += 1
            n_args = len(_split_args(text[m.end(): i - 1]))
            assert n_args == len(rs[name][1]), (fn, name, n_args, len(rs[name][1]))
            seen.add(name)
    # the seam the reference's op crates call through [compute_pipeline.rs:24-256]: the literal launch + buffers + submit
    for must in ("agpu_launch_by_name_sized", "agpu_malloc", "agpu_malloc_like", "agpu_free", "agpu_upload", "agpu_download", "agpu_copy",
                 "agpu_pipeline_create", "agpu_pipeline_finish", "agpu_pipeline_destroy", "agpu_device_create", "agpu_shader_key_for_source"):
        assert must in seen, must
    # …and the methods themselves, by the reference's names
    dev = open(os.path.join(RUST_DIR, "gpu_device.rs")).read()
    pipe = open(os.path.join(RUST_DIR, "compute_pipeline.rs")).read()
    for name in ("new", "from_adapter", "create_gpu_buffer_with_data", "create_empty_buffer", "create_retrive_buffer", "create_scalar_buffer",
                 "clone_buffer", "clone_buffer_pass", "retrive_data", "apply_unary_function", "apply_scalar_function", "apply_binary_function",
                 "apply_ternary_function", "apply_broadcast_function"):
        assert re.search(r"pub fn %s\b" % name, dev), name
    for name in ("new", "apply_unary_function", "apply_binary_function", "apply_ternary_function", "apply_scalar_function",
                 "apply_broadcast_function", "finish", "clone_buffer", "copy_buffer_to_buffer"):
        assert re.search(r"pub fn %s\b" % name, pipe), name
    assert "fn apply_take_op" in pipe and "fn apply_put_op" in pipe and "fn apply_boolean_unary_function" in pipe


def test_the_hosts_share_the_headers_limits():
    """constants the host layers repeat (the header is C, the hosts are Python / C++): they must say what include/arrow_gpu.h says"""
    import re

    from arrow_gpu_amd import _capi as capi
    from arrow_gpu_amd import gpu_utils

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "arrow_gpu.h")).read()

    def define(name):
        m = re.search(r"#define\s+" + name + r"\s+(\d+)", text)
        assert m, name
        return int(m.group(1))

    assert capi.MAILBOX_MAX_BYTES == define("AGPU_MAILBOX_MAX_BYTES")
    assert gpu_utils._CAST_CHAIN_MAX_ARRAYS == define("AGPU_CAST_CHAIN_MAX_ARRAYS")
    common = open(os.path.join(root, "arrow_gpu_amd", "csrc", "common.hpp")).read()
    slot = int(re.search(r"#define\s+AGPU_FLAG_SLOT_BYTES\s+(\d+)", common).group(1))
    payload = int(re.search(r"#define\s+AGPU_MBOX_PAYLOAD\s+(\d+)", common).group(1))
    assert slot - payload == define("AGPU_MAILBOX_MAX_BYTES")
