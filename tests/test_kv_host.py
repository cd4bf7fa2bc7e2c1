"""Host-only checks of the paged 8-bit cache's and the rotary C ABI (include/fa_kv.h, include/fa_rope.h): exports, struct
layouts, validation, workspace sizes, and the messages of the Python entry points.  No kernel is launched."""
import ctypes
import os
import re
import subprocess
import tempfile

import pytest
import torch

import torch_mlu_amd
from torch_mlu_amd import capi, capi_kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "include")
STRUCTS = [("fa_kv.h", "fa_kv_plan_params", capi_kv.FaKvPlanParams), ("fa_kv.h", "fa_kv_write_params", capi_kv.FaKvWriteParams),
           ("fa_kv.h", "fa_kv_attn_params", capi_kv.FaKvAttnParams), ("fa_rope.h", "fa_rope_params", capi_kv.FaRopeParams)]


def _stripped(header):
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, header)).read(), flags=re.S)


def test_library_exports_exactly_the_declared_symbols():
    syms = set()
    for header in ("fa_kv.h", "fa_rope.h"):
        syms |= set(re.findall(r"\b(fa_(?:kv|rope)_[a-z_]+)\s*\(", _stripped(header)))
    assert syms == set(capi_kv.EXPORTED_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", capi_kv.LIB_PATH], check=True, capture_output=True, text=True).stdout
    assert {l.split()[-1] for l in out.splitlines() if l.split()[1] in "TWVBDR"} == syms
    assert capi_kv.lib().fa_kv_version() == capi_kv.FA_KV_ABI_VERSION
    for rc in (0, -1, -2, -3, -99):
        assert capi_kv.lib().fa_kv_error_string(rc)


@pytest.mark.parametrize("header,struct,mirror", STRUCTS)
def test_ctypes_mirrors_match_the_headers(header, struct, mirror):
    names = [f[0] for f in mirror._fields_]
    text = _stripped(header)
    body = text[text.index("typedef struct " + struct):text.index("} " + struct + ";")]
    declared = [re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1]
                for stmt in body.split("{", 1)[1].split(";") if stmt.strip() for part in stmt.split(",")]
    assert declared == names
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void) {\n  printf("%%zu\\n", sizeof(%s));\n' % (header, struct)
    src += "".join('  printf("%%zu\\n", offsetof(%s, %s));\n' % (struct, n) for n in names) + "  return 0;\n}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        with open(c, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{INC}", c, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [getattr(mirror, n).offset for n in names]


def _fill(p, over, **given):
    for k, v in {**given, **over}.items():
        setattr(p, k, v)
    return p


def _plan(**over):
    """Valid blocks with made-up aligned addresses that nothing reads."""
    return _fill(capi_kv.FaKvPlanParams(), over, cached=0x1000, new_tokens=0x2000, block_table=0x3000, free_pages=0x4000, free_count=0x5000,
                 cu_seqlens=0x6000, seqused=0x7000, positions=0x8000, slots=0x9000, admitted=0xa000, free_left=0xb000, block_table_stride=20,
                 batch=4, table_pages=16, page_size=64, max_tokens=100, free_capacity=50)


def _pool(heads, D=128, page=64, block=32):
    d = dict(key_pages=0x10000, value_pages=0x20000, key_scales=0x30000, value_scales=0x40000, head_dim=D, num_pages=8, page_size=page,
             scale_block=block, dtype=capi.FA_DTYPE_BF16, format=capi_kv.FA_KV_E4M3)
    for n in ("kp", "vp"):
        d.update({n + "_stride_p": page * heads * D, n + "_stride_s": heads * D, n + "_stride_h": D})
    for n in ("ks", "vs"):
        d.update({n + "_stride_p": page // block * heads, n + "_stride_b": heads, n + "_stride_h": 1})
    return d


def _write(**over):
    d = _pool(2)
    for n in ("key", "value"):
        d.update({n + "_stride_t": 256, n + "_stride_h": 128})
    return _fill(capi_kv.FaKvWriteParams(), over, key=0x1000, value=0x2000, slots=0x3000, tokens=10, heads=2, **d)


def _attn(**over):
    d = _pool(2)
    for n in ("q", "o"):
        d.update({n + "_stride_b": 3 * 8 * 128, n + "_stride_s": 8 * 128, n + "_stride_h": 128})
    return _fill(capi_kv.FaKvAttnParams(), over, q=0x1000, out=0x2000, lse=0x3000, block_table=0x4000, seqused_k=0x5000, lse_stride_b=24,
                 lse_stride_h=3, lse_stride_s=1, block_table_stride=9, batch=2, heads_q=8, heads_k=2, seqlen_q=3, table_pages=9, scale=0.1, **d)


def _rope(**over):
    d = {}
    for n, h in (("q", 8), ("qo", 8), ("k", 2), ("ko", 2)):
        d.update({n + "_stride_b": 10 * h * 128, n + "_stride_s": h * 128, n + "_stride_h": 128})
    return _fill(capi_kv.FaRopeParams(), over, q=0x1000, k=0x2000, q_out=0x3000, k_out=0x4000, positions=0x5000, inv_freq=0x6000, axes=0x7000,
                 pos_stride_a=20, pos_stride_b=10, pos_stride_s=1, batch=2, seqlen=10, heads_q=8, heads_k=2, head_dim=128, pairs=64, num_axes=3,
                 dtype=capi.FA_DTYPE_BF16, **d)


BAD, UNS = capi.FA_ERR_BAD_ARG, capi.FA_ERR_UNSUPPORTED


@pytest.mark.parametrize("kind,make", [("fa_kv_plan", _plan), ("fa_kv_write", _write), ("fa_kv_attn", _attn), ("fa_rope", _rope)])
def test_good_blocks_pass_and_null_is_refused(kind, make):
    f = getattr(capi_kv.lib(), kind + "_validate")
    assert f(ctypes.byref(make())) == capi.FA_OK
    assert f(None) == BAD


@pytest.mark.parametrize("kind,make,over,rc", [
    ("fa_kv_plan", _plan, dict(cached=None), BAD), ("fa_kv_plan", _plan, dict(slots=0x9004), BAD), ("fa_kv_plan", _plan, dict(batch=-1), BAD),
    ("fa_kv_plan", _plan, dict(batch=8193), UNS), ("fa_kv_plan", _plan, dict(page_size=0), BAD), ("fa_kv_plan", _plan, dict(table_pages=21), BAD),
    ("fa_kv_plan", _plan, dict(table_pages=1 << 20, block_table_stride=1 << 20, page_size=1 << 12), UNS),
    ("fa_kv_plan", _plan, dict(free_pages=None), BAD), ("fa_kv_plan", _plan, dict(free_left=0x5000), BAD), ("fa_kv_plan", _plan, dict(reserved=1), BAD),
    ("fa_kv_plan", _plan, dict(seqused=0x1000), BAD), ("fa_kv_plan", _plan, dict(cu_seqlens=0x2000), BAD),
    ("fa_kv_plan", _plan, dict(max_tokens=-1), BAD), ("fa_kv_plan", _plan, dict(batch=0, cached=None, new_tokens=None, seqused=None, admitted=None), 0),
    ("fa_kv_plan", _plan, dict(free_capacity=0, free_pages=None), 0), ("fa_kv_plan", _plan, dict(max_tokens=0, slots=None, positions=None), 0),
    ("fa_kv_write", _write, dict(key=None), BAD), ("fa_kv_write", _write, dict(key=0x1008), BAD), ("fa_kv_write", _write, dict(slots=0x3004), BAD),
    ("fa_kv_write", _write, dict(value_pages=0x20008), BAD), ("fa_kv_write", _write, dict(kp_stride_s=264), BAD),
    ("fa_kv_write", _write, dict(key_stride_t=260), BAD), ("fa_kv_write", _write, dict(vs_stride_h=-1), BAD), ("fa_kv_write", _write, dict(heads=0), BAD),
    ("fa_kv_write", _write, dict(head_dim=120), UNS), ("fa_kv_write", _write, dict(head_dim=272), UNS), ("fa_kv_write", _write, dict(scale_block=16), UNS),
    ("fa_kv_write", _write, dict(scale_block=96), UNS), ("fa_kv_write", _write, dict(dtype=2), UNS), ("fa_kv_write", _write, dict(format=2), UNS),
    ("fa_kv_write", _write, dict(num_pages=1 << 25), UNS), ("fa_kv_write", _write, dict(tokens=0, key=None, value=None, slots=None), 0),
    ("fa_kv_attn", _attn, dict(q=None), BAD), ("fa_kv_attn", _attn, dict(lse=0x3002), BAD), ("fa_kv_attn", _attn, dict(block_table=None), BAD),
    ("fa_kv_attn", _attn, dict(key_scales=None), BAD), ("fa_kv_attn", _attn, dict(q_stride_s=1028), BAD), ("fa_kv_attn", _attn, dict(o_stride_b=4), BAD),
    ("fa_kv_attn", _attn, dict(batch=0), BAD), ("fa_kv_attn", _attn, dict(heads_k=3), UNS), ("fa_kv_attn", _attn, dict(is_causal=2), BAD),
    ("fa_kv_attn", _attn, dict(num_splits=65), BAD), ("fa_kv_attn", _attn, dict(table_pages=10), BAD), ("fa_kv_attn", _attn, dict(reserved=1), BAD),
    ("fa_kv_attn", _attn, dict(head_dim=8), UNS), ("fa_kv_attn", _attn, dict(kp_stride_s=1 << 26), UNS),
    ("fa_kv_attn", _attn, dict(cu_seqlens_q=0x6002, total_q=6), BAD), ("fa_kv_attn", _attn, dict(cu_seqlens_q=0x6000, total_q=-1), BAD),
    ("fa_kv_attn", _attn, dict(cu_seqlens_q=0x6000, total_q=6, q_stride_b=3), 0), ("fa_kv_attn", _attn, dict(page_size=1 << 21, scale_block=1 << 21), UNS),
    ("fa_rope", _rope, dict(q=None), BAD), ("fa_rope", _rope, dict(k=None), BAD), ("fa_rope", _rope, dict(heads_k=0, k=None, k_out=None), 0),
    ("fa_rope", _rope, dict(pairs=65), BAD), ("fa_rope", _rope, dict(pairs=0), BAD), ("fa_rope", _rope, dict(num_axes=9), UNS),
    ("fa_rope", _rope, dict(num_axes=0), BAD), ("fa_rope", _rope, dict(dtype=3), UNS), ("fa_rope", _rope, dict(head_dim=514), UNS),
    ("fa_rope", _rope, dict(positions=0x5002), BAD), ("fa_rope", _rope, dict(inv_freq=0x6004, inv_freq_64=1), BAD), ("fa_rope", _rope, dict(interleaved=2), BAD),
    ("fa_rope", _rope, dict(q=0x1002), 0), ("fa_rope", _rope, dict(q=0x1001), BAD), ("fa_rope", _rope, dict(batch=0, q=None, positions=None), 0),
])
def test_validation(kind, make, over, rc):
    L, p = capi_kv.lib(), make(**over)
    assert getattr(L, kind + "_validate")(ctypes.byref(p)) == rc
    if rc:  # launch refuses before it touches a device
        args = (None, 0, None) if kind == "fa_kv_attn" else (None,)
        assert getattr(L, kind + "_launch")(ctypes.byref(p), *args) == rc
        if kind == "fa_kv_attn":
            assert L.fa_kv_attn_workspace_bytes(ctypes.byref(p)) == 0


@pytest.mark.parametrize("kind,make,over,rc", [
    # a launch has fewer than 2^32 threads: 4 runs of up to 32 rows, or 1 to 16 tokens, a workgroup of 256
    ("fa_kv_write", _write, dict(tokens=(1 << 29) - 64), 0), ("fa_kv_write", _write, dict(tokens=1 << 29), UNS),
    ("fa_rope", _rope, dict(batch=1, seqlen=(1 << 24) - 1, q=0x1002), 0), ("fa_rope", _rope, dict(batch=1, seqlen=1 << 24, q=0x1002), UNS),
    ("fa_rope", _rope, dict(batch=1, seqlen=1 << 24, heads_q=1, heads_k=0), 0), ("fa_rope", _rope, dict(batch=1, seqlen=1 << 28, heads_q=1, heads_k=0), UNS),
])
def test_calls_beyond_one_launch_are_refused(kind, make, over, rc):
    L, p = capi_kv.lib(), make(**over)
    assert getattr(L, kind + "_validate")(ctypes.byref(p)) == rc
    if rc:
        assert getattr(L, kind + "_launch")(ctypes.byref(p), None) == rc


@pytest.mark.parametrize("over", [dict(batch=1 << 25, num_splits=1), dict(batch=1 << 20, seqlen_q=1 << 10, num_splits=1),
                                  dict(cu_seqlens_q=0x6000, total_q=1 << 30, seqlen_q=1 << 20, num_splits=1)])
def test_attention_beyond_one_launch_is_refused(over):
    p = _attn(**over)  # refused before it touches a device
    assert capi_kv.lib().fa_kv_attn_launch(ctypes.byref(p), None, 0, None) == UNS


def test_attention_workspace():
    """Partial results (an fp32 row, its maximum and sum) of every query row and slice; short workspaces are refused."""
    L = capi_kv.lib()
    one = _attn(num_splits=1)
    assert L.fa_kv_attn_workspace_bytes(ctypes.byref(one)) == 0
    p = _attn(num_splits=5)
    need = L.fa_kv_attn_workspace_bytes(ctypes.byref(p))
    assert need == 2 * 8 * 3 * 5 * (128 * 4 + 8)
    assert L.fa_kv_attn_launch(ctypes.byref(p), None, 0, None) == BAD
    assert L.fa_kv_attn_launch(ctypes.byref(p), 0x7000, need - 1, None) == BAD
    assert L.fa_kv_attn_launch(ctypes.byref(p), 0x7008, need, None) == BAD
    few = _attn(num_splits=64, table_pages=1)  # never more slices than 32-key blocks
    assert L.fa_kv_attn_workspace_bytes(ctypes.byref(few)) == 2 * 8 * 3 * 2 * (128 * 4 + 8)


def test_python_entry_points_refuse_what_is_not_on_the_device():
    z = torch.zeros
    i = lambda *s: z(s, dtype=torch.int32)  # noqa: E731
    f8 = z(4, 64, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = z(4, 2, 2)
    for call in (lambda: torch_mlu_amd.paged_plan(i(2), i(2), i(2, 4), i(9), i(1), page_size=64, max_tokens=8),
                 lambda: torch_mlu_amd.paged_cache_write(z(3, 2, 64, dtype=torch.half), z(3, 2, 64, dtype=torch.half), f8, f8, sc, sc, z(3, dtype=torch.int64)),
                 lambda: torch_mlu_amd.paged_attention(z(2, 4, 1, 64, dtype=torch.half), f8, f8, i(2, 2), i(2), key_scales=sc, value_scales=sc),
                 lambda: torch_mlu_amd.rotary(z(1, 2, 3, 8), None, i(1, 3), *torch_mlu_amd.rotary_frequencies((4,)))):
        with pytest.raises(RuntimeError, match="Input tensor must be on HIP device"):
            call()
    with pytest.raises(ValueError, match="go together"):
        torch_mlu_amd.paged_attention(z(2, 4, 1, 64), f8, f8, i(2, 2), i(2), key_scales=sc)
    with pytest.raises(ValueError, match="packed queries need a cache in 8 bits"):
        torch_mlu_amd.paged_attention(z(2, 4, 64), z(4, 64, 2, 64), z(4, 64, 2, 64), i(2, 2), i(2), cu_seqlens_q=i(3), max_seqlen_q=1)
    with pytest.raises(ValueError, match="needs key_scales"):
        torch_mlu_amd.paged_attention(z(2, 4, 1, 64), f8, f8, i(2, 2), i(2))


def test_rotary_frequencies():
    f, a = torch_mlu_amd.rotary_frequencies((2, 1, 1), theta=16.0)
    assert f.tolist() == [1.0, 0.5, 0.25, 0.125] and a.tolist() == [0, 0, 1, 2] and f.dtype == torch.float64 and a.dtype == torch.int32
    f, a = torch_mlu_amd.rotary_frequencies((2, 2), theta=16.0, per_axis=True)
    assert f.tolist() == [1.0, 0.25, 1.0, 0.25] and a.tolist() == [0, 0, 1, 1]
    for bad in ((), (0,), (2, -1)):
        with pytest.raises(ValueError):
            torch_mlu_amd.rotary_frequencies(bad)


def test_host_half_is_clean_under_asan_and_ubsan():
    """Validation, plans and workspace sizes (csrc/fa_kv_host.h) over ordinary, extreme and malformed blocks, built with the address and
    undefined-behaviour sanitizers: any overflow or out-of-bounds access ends the driver."""
    import shutil

    if shutil.which("g++") is None:
        pytest.skip("no host C++ compiler")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "kv_host_sanitize")
        subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-static-libasan", "-fno-sanitize-recover=all", "-Wall", "-Werror",
                        "-I" + INC, "-I" + os.path.join(ROOT, "torch_mlu_amd", "csrc"), os.path.join(ROOT, "tests", "kv_host_sanitize.cpp"), "-o", exe],
                       check=True)
        res = subprocess.run([exe], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    assert re.match(r"\d+ blocks, \d+ plans", res.stdout)
