"""Host side of the token-step operators: refusals (before any GPU work, so they hold on a machine
without one), the weight packer, the cache struct and the ABI's Python mirror."""
import ctypes as C
import os

import numpy as np
import pytest

from sys1rust_b200 import backend as bk
from sys1rust_b200 import operators as ops
from sys1rust_b200.backend import BackendError

BUF = np.zeros(4096, dtype=np.uint8)
PTR = (BUF.ctypes.data + 255) // 256 * 256  # never read: every call below is refused


def _refused(call, *args, text="", **kw):
    with pytest.raises(BackendError) as e:
        call(*args, **kw)
    assert e.value.code == bk.S1C_ERR_ARG
    assert text in str(e.value)


def _nibble(**kw):
    a = dict(dtype=ops.DT_BF16, x_ptr=PTR, x_stride=64, codes_ptr=PTR, code_pitch=32, scales_ptr=PTR, scale_stride=2,
             out_ptr=PTR, out_stride=8, M=1, N=8, K=64, group=32)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=ops.DT_F32), "dtype"), (dict(dtype=7), "dtype"), (dict(x_ptr=0), "null"), (dict(codes_ptr=0), "null"),
    (dict(scales_ptr=0), "null"), (dict(out_ptr=0), "null"), (dict(M=65), "M must"), (dict(M=-1), "M must"), (dict(N=(1 << 30) + 1), "M must"),
    (dict(N=0), "M must"), (dict(K=0), "M must"), (dict(group=48), "group"), (dict(group=0), "group"),
    (dict(code_pitch=24), "pitch"), (dict(code_pitch=16), "pitch"), (dict(codes_ptr=PTR + 8), "aligned"),
    (dict(x_stride=63), "stride"), (dict(out_stride=7), "stride"), (dict(scale_stride=1), "stride"), (dict(act=3), "act"),
    (dict(act=-1), "act")])
def test_nibble_gemm_refuses(bad, text):
    _refused(ops.nibble_gemm, text=text, **_nibble(**bad))


def _cache(**kw):
    a = dict(k_codes_ptr=PTR, v_codes_ptr=PTR, k_scales_ptr=PTR, v_scales_ptr=PTR, num_pages=4, page=16, kv_heads=2,
             head_dim=64)
    a.update(kw)
    return ops.Cache(**a)


BAD_CACHES = [(dict(k_codes_ptr=0), "null"), (dict(v_codes_ptr=0), "null"), (dict(k_scales_ptr=0), "null"),
              (dict(v_scales_ptr=0), "null"), (dict(num_pages=0), "num_pages"), (dict(kv_heads=0), "kv_heads"),
              (dict(kv_heads=70000), "kv_heads"), (dict(page=8), "page"), (dict(page=48), "page"),
              (dict(head_dim=96), "head_dim"), (dict(k_codes_ptr=PTR + 4), "aligned"), (dict(num_pages=1 << 30), "2^31")]


def _rows(**kw):
    a = dict(cache=_cache(), dtype=ops.DT_F16, k_ptr=PTR, k_stride=128, v_ptr=PTR, v_stride=128, cu_ptr=PTR, start_ptr=PTR,
             pages_ptr=PTR, max_pages=2, n=1)
    a.update(kw)
    return a


BAD_ROWS = [(dict(dtype=ops.DT_F32), "dtype"), (dict(k_ptr=0), "null"), (dict(v_ptr=0), "null"), (dict(cu_ptr=0), "null"),
            (dict(start_ptr=0), "null"), (dict(pages_ptr=0), "null"), (dict(k_stride=120), "stride"),
            (dict(v_stride=129), "stride"), (dict(k_ptr=PTR + 2), "aligned"), (dict(v_ptr=PTR + 8), "aligned"),
            (dict(max_pages=0), "max_pages"), (dict(n=-1), "negative")]


@pytest.mark.parametrize("bad,text", BAD_CACHES)
def test_cache_calls_refuse_a_bad_cache(bad, text):
    c = _cache(**bad)
    _refused(ops.cache_write, text=text, max_new=1, **_rows(cache=c))
    _refused(ops.cache_read, text=text, max_rows=1, **_rows(cache=c))
    _refused(ops.cache_attention, text=text, **_attend(cache=c))


@pytest.mark.parametrize("bad,text", BAD_ROWS + [(dict(max_new=-1), "negative"), (dict(n=1 << 30, max_new=1 << 30), "2^31")])
def test_cache_write_refuses(bad, text):
    _refused(ops.cache_write, text=text, **_rows(**{"max_new": 1, **bad}))


@pytest.mark.parametrize("bad,text", BAD_ROWS + [(dict(max_rows=-1), "negative"), (dict(n=1 << 30, max_rows=1 << 30), "large")])
def test_cache_read_refuses(bad, text):
    _refused(ops.cache_read, text=text, **_rows(**{"max_rows": 1, **bad}))


def _attend(**kw):
    a = dict(cache=_cache(), dtype=ops.DT_BF16, q_ptr=PTR, q_stride=256, out_ptr=PTR, out_stride=256, heads=4, cu_ptr=PTR,
             len_ptr=PTR, pages_ptr=PTR, max_pages=2, n=1, max_q=1, max_kv=32, scale=0.125, workspace_ptr=PTR,
             workspace_bytes=1 << 40)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=ops.DT_F32), "dtype"), (dict(q_ptr=0), "null"), (dict(out_ptr=0), "null"), (dict(cu_ptr=0), "null"),
    (dict(len_ptr=0), "null"), (dict(pages_ptr=0), "null"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
    (dict(q_stride=248), "stride"), (dict(out_stride=260), "stride"), (dict(q_ptr=PTR + 8), "aligned"),
    (dict(out_ptr=PTR + 2), "aligned"), (dict(n=-1), "negative"), (dict(max_q=-1), "negative"), (dict(max_kv=-1), "negative"),
    (dict(max_pages=0), "max_pages"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(n=1 << 20, max_q=1 << 20), "2^31")])
def test_cache_attention_refuses(bad, text):
    _refused(ops.cache_attention, text=text, **_attend(**bad))


def test_cache_attention_refuses_a_short_workspace():
    need = ops.cache_attention_workspace(_cache(), 4, 1, 1, 100000)
    if need:
        _refused(ops.cache_attention, text="workspace", **_attend(max_kv=100000, workspace_bytes=need - 1))
        _refused(ops.cache_attention, text="workspace", **_attend(max_kv=100000, workspace_ptr=0, workspace_bytes=need))
        _refused(ops.cache_attention, text="workspace", **_attend(max_kv=100000, workspace_ptr=PTR + 4, workspace_bytes=need))
    assert ops.cache_attention_workspace(_cache(page=5), 4, 1, 1, 100000) == 0  # a cache that the call refuses
    assert bk.lib().s1c_cache_attention_workspace(None, 4, 1, 1, 100000) == 0


def test_cache_attention_workspace_of_refused_bounds_is_zero():
    big = 2 ** 31 - 1
    for bounds in [(4, big, big, 4096), (4, 1, 1, big), (2 ** 30, 4, 1, 4096), (4, 1, big, 4096), (4, 0, 1, 4096), (3, 1, 1, 4096)]:
        assert ops.cache_attention_workspace(_cache(), *bounds) == 0, bounds
    assert ops.cache_attention_workspace(_cache(), 4, 2 ** 15, 2 ** 13, 2 ** 30) > 2 ** 50  # the largest: no overflow


@pytest.mark.parametrize("heads,kv_heads,page,dim", [(8, 8, 16, 64), (32, 8, 16, 128), (4, 4, 64, 128), (80, 2, 32, 64),
                                                     (16, 1, 16, 128)])
def test_cache_attention_workspace_serves_smaller_calls(heads, kv_heads, page, dim):
    """The workspace of some bounds is accepted by every call with smaller ones, however these split their keys; sizes
    next to those at which the split changes are among them. The calls stop at their host memory, behind the check."""
    c = _cache(kv_heads=kv_heads, head_dim=dim, page=page)
    rng = np.random.default_rng(5)
    kvs = [1, 128, 129, 2048, 2049, 256 * page - 128, 256 * page - 127, 30000, 131072]
    qs = sorted({1, 2, 32 * kv_heads // heads or 1, 32 * kv_heads // heads + 1, 128, 500})

    def call(n, q, kv, size):
        with pytest.raises(BackendError) as e:
            ops.cache_attention(**_attend(cache=c, heads=heads, q_stride=heads * dim, out_stride=heads * dim, n=n, max_q=q, max_kv=kv,
                                          workspace_bytes=size))
        return str(e.value)

    for n, q, kv in [(64, 1, 2048), (64, 1, 8192), (37, 1, 131072), (4, 500, 4000), (300, 40, 5000), (148, 128, 3968), (1, 1, 200)]:
        size = ops.cache_attention_workspace(c, heads, n, q, kv)
        # what the call itself checks for
        if size:
            short = call(n, q, kv, size - 1)
            assert "workspace" in short or "workspace" not in call(n, q, kv, 0)  # a call that needs none takes none
        assert "workspace" not in call(n, q, kv, size)
        smaller = [(a, b, k) for a in (1, 2, 3, 5, 18, 19, 55, 56, 64, 148) for b in qs for k in kvs]
        for a, b, k in [smaller[i] for i in rng.permutation(len(smaller))[:150]] + [(1, 1, kv), (1, q, kv), (n // 2, q, kv // 2)]:
            a, b, k = max(1, min(a, n)), min(b, q), max(1, min(k, kv))
            assert ops.cache_attention_workspace(c, heads, a, b, k) <= size, (a, b, k)
            assert "workspace" not in call(a, b, k, size), (a, b, k)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), "dtype"), (dict(logits_ptr=0), "null"), (dict(uniform_ptr=0), "null"), (dict(token_ptr=0), "null"),
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1, row_stride=1 << 22), "vocab"),
    (dict(row_stride=9), "stride")])
def test_sample_refuses(bad, text):
    a = dict(dtype=ops.DT_F32, logits_ptr=PTR, row_stride=10, rows=1, vocab=10, token_ptr=PTR, uniform_ptr=PTR)
    a.update(bad)
    _refused(ops.sample, text=text, **a)


def test_pointers_off_their_element_type_are_refused():
    """An odd address of 16-bit elements, or one off by two of 32-bit ones, would fault on the GPU."""
    bad = dict(text="element type")
    for name, by in [("x_ptr", 1), ("scales_ptr", 1), ("zeros_ptr", 1), ("bias_ptr", 2), ("out_ptr", 1)]:
        _refused(ops.nibble_gemm, **bad, **_nibble(**{name: PTR + by}))
    _refused(ops.nibble_gemm, **bad, **_nibble(out_ptr=PTR + 2, out_f32=True))
    for name in ("k_scales_ptr", "v_scales_ptr"):
        c = _cache(**{name: PTR + 2})
        _refused(ops.cache_write, max_new=1, **bad, **_rows(cache=c))
        _refused(ops.cache_read, max_rows=1, **bad, **_rows(cache=c))
        _refused(ops.cache_attention, **bad, **_attend(cache=c))
    for name in ("cu_ptr", "start_ptr", "pages_ptr"):
        _refused(ops.cache_write, max_new=1, **bad, **_rows(**{name: PTR + 2}))
        _refused(ops.cache_read, max_rows=1, **bad, **_rows(**{name: PTR + 2}))
    for name in ("lse_ptr", "cu_ptr", "len_ptr", "pages_ptr"):
        _refused(ops.cache_attention, **bad, **_attend(**{name: PTR + 2}))
    a = dict(dtype=ops.DT_F32, logits_ptr=PTR, row_stride=10, rows=1, vocab=10, token_ptr=PTR, uniform_ptr=PTR)
    for name in ("logits_ptr", "token_ptr", "uniform_ptr", "temperature_ptr", "top_k_ptr", "top_p_ptr", "min_p_ptr", "prob_ptr"):
        _refused(ops.sample, **bad, **{**a, name: PTR + 2})
    _refused(ops.sample, **bad, **{**a, "dtype": ops.DT_BF16, "logits_ptr": PTR + 1})


def test_nibble_pack_refuses_scales_that_do_not_fit():
    with pytest.raises(BackendError):
        ops.nibble_pack(np.full((1, 32), 1e6), 32, scale_dtype=np.float16)  # 142857 is past f16


def test_calls_without_rows_do_nothing():
    """No rows: accepted without touching the GPU."""
    ops.nibble_gemm(**_nibble(M=0))
    ops.cache_write(max_new=1, **_rows(n=0))
    ops.cache_write(max_new=0, **_rows())
    ops.cache_read(max_rows=0, **_rows())
    ops.cache_attention(**_attend(n=0))
    ops.cache_attention(**_attend(max_q=0))
    ops.sample(ops.DT_F32, PTR, 10, 0, 10, PTR, PTR)


def test_nibble_pack_round_trip():
    """Each weight comes back within half a step of its group's scale; padding columns hold zero."""
    rng = np.random.default_rng(1)
    for N, K, group in [(3, 64, 32), (5, 100, 64), (2, 1, 128), (4, 261, 128)]:
        w = rng.standard_normal((N, K)).astype(np.float32)
        w[0, : min(K, 10)] = 0
        codes, scales = ops.nibble_pack(w, group)
        assert codes.shape == (N, -(-K // 32) * 16) and scales.shape == (N, -(-K // group))
        q = np.stack([codes & 15, codes >> 4], -1).reshape(N, -1).astype(np.int64) - 8
        assert (q[:, K:] == 0).all() and q.min() >= -7
        s = scales.astype(np.float64)[:, np.arange(K) // group]
        # half a step, and the rounding of w / scale in the packer's 64 bits
        assert (np.abs(q[:, :K] * s - w) <= s * (0.5 + 1e-6)).all()
    for bad in [np.zeros((2, 2, 2)), np.full((2, 32), np.nan)]:
        with pytest.raises(BackendError):
            ops.nibble_pack(bad, 32)
    with pytest.raises(BackendError):
        ops.nibble_pack(np.zeros((2, 32)), 16)


def test_cache_struct_matches_the_header(tmp_path):
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = [f for f, _ in bk.CCache._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "s1c.h"\nint main(void) {\n  printf("%zu", sizeof(s1c_cache));\n' +
                   "".join(f'  printf(" %zu", offsetof(s1c_cache, {n}));\n' for n in names) + "  return 0;\n}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([cc, "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(bk.CCache)] + [getattr(bk.CCache, n).offset for n in names]


def test_kernels_hold_their_tmem_before_a_successor_may_start():
    """A kernel that is scheduled early can hold tensor memory while it waits for its predecessor. If a block of the
    predecessor had still to allocate its own, neither would end: so each kernel calls pdl_trigger after its
    allocation and a barrier of the block (attn_pages has some)."""
    import re
    csrc = os.path.join(os.path.dirname(os.path.abspath(bk.__file__)), "csrc")
    checked = []
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for body in re.split(r"__global__", text)[1:]:
            alloc = re.search(r"\btmem_alloc2?\(", body)
            if alloc:
                trigger = re.search(r"\bpdl_trigger\(\)", body)
                assert trigger is None or alloc.start() < trigger.start(), name
                assert trigger is None or re.search("__syncthreads|cluster_sync_all|attn_pages", body[alloc.end(): trigger.start()]), name
                checked.append(name)
    assert "cache_attention.cuh" in checked and "gemm_sm100_csk.cuh" in checked


def test_attention_timeout_selftest_checks_its_arguments():
    for budget in (0, 10, 3 * 10 ** 9):
        with pytest.raises(BackendError):
            bk.selftest_cache_attention_timeout(0, budget)
    assert bk.lib().s1c_selftest_cache_attention_timeout(0, 10 ** 7, None) == bk.S1C_ERR_ARG
