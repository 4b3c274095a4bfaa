"""The token-step operators on the GPU against plain computations in 64 bits.

Tolerances, derived: storing a result of type t is off by at most u_t = eps_t / 2 of it (bf16 2^-8, f16 2^-11,
fp32 2^-24). A sum of K products held in fp32, in any order and with truncating adders (at most 2^-23
a step), is off by at most K 2^-22 of the sum of the products' magnitudes. Where a bound has more
parts, the test that uses it names them.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from sys1rust_b200 import operators
    return operators


def _code(ops, dt):
    return {torch.bfloat16: ops.DT_BF16, torch.float16: ops.DT_F16, torch.float32: ops.DT_F32}[dt]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------
# products with 4-bit weights


def _nibble_inputs(M, N, K, group, dt, zeros, seed, pad=0):
    g = _gen(seed)
    pitch = -(-K // 32) * 16 + 16 * pad
    groups = -(-K // group)
    x = torch.randn(M, K + 3 * pad, generator=g, device="cuda").to(dt)[:, :K]
    codes = torch.randint(0, 256, (N, pitch), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(N, groups + pad, generator=g, device="cuda") + 0.25).to(dt)[:, :groups]
    z = (torch.rand(N, groups + pad, generator=g, device="cuda") * 15).to(dt)[:, :groups] if zeros else None
    return x, codes, scales, z


def _nibble_weights(codes, scales, zeros, K, group):
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :K].double()
    at = torch.arange(K, device="cuda") // group
    return (q - (zeros.double()[:, at] if zeros is not None else 8.0)) * scales.double()[:, at]


def _nibble(ops, x, codes, scales, zeros, out, K, group, bias=None, act=0, stream=None):
    M, N = out.shape
    ops.nibble_gemm(_code(ops, x.dtype), x.data_ptr(), x.stride(0), codes.data_ptr(), codes.stride(0), scales.data_ptr(),
                    scales.stride(0), out.data_ptr(), out.stride(0), M, N, K, group, zeros_ptr=_ptr(zeros),
                    bias_ptr=_ptr(bias), act=act, out_f32=out.dtype == torch.float32, stream=_stream() if stream is None else stream)


def _act(y, act):
    return y if act == 0 else torch.relu(y) if act == 1 else torch.nn.functional.gelu(y)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K,group", [
    (1, 1, 1, 32), (1, 7, 31, 32), (2, 16, 32, 64), (1, 64, 33, 128), (1, 1024, 1024, 128), (3, 130, 257, 32),
    (5, 1000, 2624, 64), (8, 33, 4097, 128), (9, 300, 640, 32), (16, 257, 1100, 64), (17, 129, 129, 128), (33, 65, 2047, 32),
    (64, 200, 1024, 128), (64, 31, 5000, 64), (1, 5000, 96, 32), (4, 20000, 160, 64), (2, 48, 20000, 128),
    (8, 100, 9000, 32), (16, 70, 6001, 64), (12, 300, 8192, 128), (6, 40, 30000, 64), (3, 2400, 12000, 128),
    (45, 70, 9000, 32), (64, 20, 16000, 128), (20, 50, 2700, 64), (10, 17, 100000, 32), (1, 33, 90001, 128),
    (17, 40, 9900, 64)])
def test_nibble_gemm(ops, M, N, K, group, dt):
    """Every combination of zero points, bias, activation and output type at one or another size. The
    error is the sum's, the zero point's and bias's place in it, and one rounding; GELU's slope is at most 1.13."""
    for i, (zeros, bias, act, f32) in enumerate([(False, False, 0, False), (True, True, 0, True), (True, False, 1, False),
                                                 (False, True, 2, True), (True, True, 2, False)]):
        x, codes, scales, z = _nibble_inputs(M, N, K, group, DT[dt], zeros, 100 + i, pad=i % 2)
        b = torch.randn(N, generator=_gen(7), device="cuda") if bias else None
        odt = torch.float32 if f32 else DT[dt]
        full = torch.full((M, N + 5), 7.0, dtype=odt, device="cuda")
        out = full[:, :N]
        _nibble(ops, x, codes, scales, z, out, K, group, b, act)
        w = _nibble_weights(codes, scales, z, K, group)
        y = x.double() @ w.t() + (b.double() if bias else 0)
        ref = _act(y, act)
        # codes and zero points stand apart in the sum: |q| + |z| up to 30 a product, times the scale
        at = torch.arange(K, device="cuda") // group
        mag = x.double().abs() @ (scales.double()[:, at] * 30).t() + (b.double().abs() if bias else 0)
        bound = _u(odt) * ref.abs() + 1.13 * (K + 64) * 2.0 ** -22 * mag + torch.finfo(odt).tiny
        err = (out.double() - ref).abs()
        assert (err <= bound).all(), (i, (err / bound).max().item())
        assert (full[:, N:] == 7).all()


@pytest.mark.parametrize("M,N,K,group", [(64, 33, 9000, 128), (9, 16, 300, 32), (9, 33, 300, 64), (11, 17, 1000, 128),
                                         (64, 50, 300, 128), (55, 2400, 8000, 32), (17, 3000, 700, 64)])
def test_nibble_gemm_staged_by_two_blocks(ops, M, N, K, group):
    """From nine rows on two blocks stage x together: one row tile (a block alone), odd numbers of rows and
    tiles, several launches whose last has few rows. Bounds as in test_nibble_gemm."""
    test_nibble_gemm(ops, M, N, K, group, "bf16")


def test_nibble_gemm_extreme_codes_and_values(ops):
    """All codes 0 or 15 with the largest finite x of f16 in fp32 output; zero scales give zero; a NaN or
    infinite row of x stays in its own row; bytes behind the last column do not count."""
    M, N, K, group = 3, 40, 200, 32
    x, codes, scales, _ = _nibble_inputs(M, N, K, group, torch.float16, False, 5)
    codes[:20] = 0
    codes[20:] = 255
    codes[:, 100:] = 0x5A  # behind column 200
    x[0] = 65504.0
    scales[3] = 0
    out = torch.empty(M, N, device="cuda")
    _nibble(ops, x, codes, scales, None, out, K, group)
    w = _nibble_weights(codes, scales, None, K, group)
    ref = x.double() @ w.t()
    bound = (K + 64) * 2.0 ** -22 * (x.double().abs() @ (scales.double()[:, torch.arange(K, device="cuda") // group] * 30).t()) + 1e-30
    assert ((out.double() - ref).abs() <= bound).all()
    assert (out[:, 3] == 0).all()
    x2 = x.clone()
    x2[1, 7] = float("nan")
    x2[2, 0] = float("inf")
    out2 = torch.empty_like(out)
    _nibble(ops, x2, codes, scales, None, out2, K, group)
    assert torch.equal(out2[0], out[0])
    keep = torch.arange(N, device="cuda") != 3
    assert torch.isnan(out2[1][keep]).all() and not torch.isfinite(out2[2][keep]).any()


def test_nibble_gemm_rows_far_from_one(ops):
    """bf16 rows from 2^-124 (subnormal values among them) to 2^120 keep the bound of the sum: the rows' scaling and
    its undoing leave the range of fp32 nowhere; with few columns, in several launches, and in pieces."""
    for K, rows in [(256, 7), (9000, 7), (100000, 7)]:
        x, codes, scales, _ = _nibble_inputs(rows, 40, K, 128, torch.bfloat16, False, 9)
        for m, p in enumerate([-124, -120, -112, -90, -40, 40, 110]):
            x[m] = (x[m].double() * 2.0 ** p).to(torch.bfloat16)
        out = torch.empty(rows, 40, device="cuda")
        _nibble(ops, x, codes, scales, None, out, K, 128)
        ref = x.double() @ _nibble_weights(codes, scales, None, K, 128).t()
        mag = x.double().abs() @ (scales.double()[:, torch.arange(K, device="cuda") // 128] * 30).t()
        # as in test_nibble_gemm; results below the normal range are stored to 2^-149
        bound = (K + 64) * 2.0 ** -22 * mag + _u(torch.float32) * ref.abs() + 2.0 ** -149
        err = (out.double() - ref).abs()
        assert (err <= bound).all(), (K, (err / bound).max(1).values)


def test_nibble_gemm_is_bitwise_repeatable_and_row_independent(ops):
    """The same call gives the same bits; the packer's codes give its weights' products."""
    x, codes, scales, z = _nibble_inputs(7, 515, 3001, 64, torch.bfloat16, True, 9)
    outs = []
    for _ in range(2):
        out = torch.empty(7, 515, device="cuda")
        _nibble(ops, x, codes, scales, z, out, 3001, 64)
        outs.append(out)
    assert torch.equal(*outs)
    w = torch.randn(50, 300, generator=torch.Generator().manual_seed(3)).numpy()
    packed, s = ops.nibble_pack(w, 64, np.float16)
    packed, s = torch.from_numpy(packed).cuda(), torch.from_numpy(s).cuda()
    xs = torch.randn(2, 300, generator=_gen(4), device="cuda").half()
    out = torch.empty(2, 50, device="cuda")
    _nibble(ops, xs, packed, s, None, out, 300, 64)
    # each weight is off by at most half a step (and the scale's f16 rounding within it, clipped at 7)
    step = s.double()[:, torch.arange(300, device="cuda") // 64]
    ref = xs.double() @ torch.from_numpy(w).cuda().double().t()
    assert ((out.double() - ref).abs() <= xs.double().abs() @ (0.51 * step).t() + 1e-3).all()


WIDE = [(1, 70, 90001, 128), (10, 17, 100000, 32), (3, 300, 120001, 64), (8, 33, 300000, 128), (64, 31, 5000, 64), (45, 70, 9000, 32),
        (64, 50, 16000, 128), (17, 129, 9900, 64), (8, 100, 9000, 32), (16, 70, 6001, 64), (12, 300, 8192, 128), (6, 40, 30000, 64),
        (3, 2400, 12000, 128), (1, 5000, 2624, 64), (33, 260, 2047, 32)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", WIDE)
def test_nibble_gemm_whole_numbers_are_exact(ops, M, N, K, group, zeros, dt):
    """Whole x, scales that are powers of two and whole zero points: every sum is a multiple of a half below
    2^23, so the result is exact in whatever order it is formed, and equal to the definition's. One row has larger values
    in its second half and one zeros in its first, so that the scaling of rows whose x passes in blocks of columns
    changes on the way."""
    g = _gen(K + M)
    x = torch.randint(-1, 2, (M, K), generator=g, device="cuda").double()
    some = torch.rand(M, K, generator=g, device="cuda") < 1 / 128
    half = torch.arange(K, device="cuda") >= K // 2
    if M > 1:
        x[M // 2] = torch.where(half & some[0], x[M // 2] * 32, torch.where(some[1], x[M // 2], 0.0))
    x[M - 1] *= half
    _, codes, _, _ = _nibble_inputs(1, N, K, group, DT[dt], False, K)
    groups = -(-K // group)
    scales = torch.exp2(torch.randint(-1, 2, (N, groups), generator=g, device="cuda").double()).to(DT[dt])
    z = torch.randint(0, 16, (N, groups), generator=g, device="cuda").to(DT[dt]) if zeros else None
    if K > 100000:  # keep to 2^23
        x *= torch.rand(M, K, generator=g, device="cuda") < 100000 / K / 3
    w = _nibble_weights(codes, scales, z, K, group)
    # q and z stand apart in a group's sum; each is at most 15
    at = torch.arange(K, device="cuda") // group
    assert (x.abs() @ scales.double()[:, at].t()).max() * 30 * 2 < 2 ** 24
    out = torch.empty(M, N, device="cuda")
    _nibble(ops, x.to(DT[dt]), codes, scales, z, out, K, group)
    want = x @ w.t()
    assert torch.equal(out.double(), want), (out.double() - want).abs().max()
    assert (want != 0).double().mean() > 0.9


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K,group", WIDE)
def test_nibble_gemm_wide_rows(ops, M, N, K, group, dt):
    """Any values, with a bound that stays far below the result however wide the rows are. A group's sum takes `group`
    products and its first value, each off by at most 2^-23 of the magnitudes in the group (truncating adders),
    and x loses at most 2^-35 of its row's largest; the groups' results, and the pieces of a tile, then add up with one rounding
    each, of 2^-24 of a sum of neighbouring groups, which is at most twice the largest of the running sums."""
    x, codes, scales, z = _nibble_inputs(M, N, K, group, DT[dt], True, 17)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :K].double()
    groups = -(-K // group)
    pad = groups * group - K
    xs, qs = [torch.nn.functional.pad(t, (0, pad)).view(-1, groups, group) for t in (x.double(), q)]
    s, zz = scales.double(), z.double()
    part = s * (torch.einsum("mgk,ngk->mng", xs, qs) - zz * xs.sum(2)[:, None])
    mag = s * (torch.einsum("mgk,ngk->mng", xs.abs(), qs) + zz * xs.abs().sum(2)[:, None])
    ref = part.sum(2)
    run = torch.nn.functional.pad(part.cumsum(2), (1, 0))
    spread = run.amax(2) - run.amin(2)
    bound = (group + 16) * 2.0 ** -23 * mag.sum(2) + 2 * (groups + 40) * 2.0 ** -24 * spread + _u(torch.float32) * ref.abs()
    out = torch.empty(M, N, device="cuda")
    _nibble(ops, x, codes, scales, z, out, K, group)
    err = (out.double() - ref).abs()
    assert (err <= bound).all(), (err / bound).max()
    assert bound.mean() < 0.05 * ref.abs().mean()  # so that a wrong result fails


@pytest.mark.parametrize("M,N,K,group", [(7, 515, 3001, 64), (16, 100, 2624, 128), (40, 64, 9000, 32), (8, 40, 100000, 64)])
def test_nibble_gemm_rows_do_not_depend_on_each_other(ops, M, N, K, group):
    """A row's bits are the same whatever the other rows of the call hold."""
    x, codes, scales, z = _nibble_inputs(M, N, K, group, torch.bfloat16, True, 19)
    outs = []
    for by in (1.0, 1e4, math.nan):
        y = x.clone()
        y[::3] *= by
        out = torch.empty(M, N, device="cuda")
        _nibble(ops, y, codes, scales, z, out, K, group)
        outs.append(out)
    keep = torch.arange(M, device="cuda") % 3 != 0
    assert torch.equal(outs[0][keep], outs[1][keep]) and torch.equal(outs[0][keep], outs[2][keep])
    assert not torch.equal(outs[0], outs[1]) and torch.isnan(outs[2][~keep]).all()


def test_nibble_gemm_codes_past_four_gigabytes(ops):
    """A matrix of 4.6 GB of codes with rows of x and out past 2^31 elements: its first and last rows."""
    M, N, K, group = 3, 1150000, 8000, 128
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    g = _gen(23)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-1, 2, (N, 63), generator=g, device="cuda").float()).half()
    stride = 2 ** 30 + 4
    x = torch.empty(2 * stride + K, dtype=torch.float16, device="cuda").as_strided((M, K), (stride, 1))
    x.copy_(torch.randint(-1, 2, (M, K), generator=g, device="cuda"))
    out = torch.empty(2 * stride + N, dtype=torch.float32, device="cuda").as_strided((M, N), (stride, 1))
    _nibble(ops, x, codes, scales, None, out, K, group)
    for rows in (slice(0, 100), slice(N // 2, N // 2 + 100), slice(N - 100, N)):
        want = x.double() @ _nibble_weights(codes[rows], scales[rows], None, K, group).t()
        assert torch.equal(out[:, rows].double(), want)


# ---------------------------------------------------------------------------------------------
# the cache


class Paged:
    """A cache on the GPU and the values it should hold, kept by a plain computation in 64 bits."""

    def __init__(self, ops, n, longest, H, D, page, seed, spare=3):
        per = -(-longest // page)
        self.count = n * per + spare
        g = _gen(seed)
        self.H, self.D, self.page, self.n, self.ops = H, D, page, n, ops
        self.table = torch.randperm(self.count, generator=g, device="cuda")[: n * per].view(n, per).to(torch.int32).contiguous()
        shape = (self.count, H, page, D)
        self.codes = [torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
        self.scales = [torch.rand(self.count, H, generator=g, device="cuda") * 0.02 + 0.01 for _ in range(2)]
        self.handle = ops.Cache(self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(),
                                self.scales[1].data_ptr(), self.count, page, H, D)
        self.expect()

    def expect(self):
        self.want_codes = [c.double().cpu() for c in self.codes]
        self.want_scales = [s.double().cpu() for s in self.scales]

    def write(self, k, v, lens, starts, most=None):
        cu = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
        st = _i32(starts)
        self.ops.cache_write(self.handle, _code(self.ops, k.dtype), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                             cu.data_ptr(), st.data_ptr(), self.table.data_ptr(), self.table.shape[1], self.n,
                             max(lens) if most is None else most, stream=_stream())
        torch.cuda.synchronize()
        table = self.table.cpu()
        for which, x in enumerate((k, v)):
            x = x.double().cpu().view(x.shape[0], self.H, self.D)
            base = 0
            for i, (c, a) in enumerate(zip(lens, starts)):
                c2 = c if most is None else min(c, most)
                for p in range(a // self.page, -(-(a + c2) // self.page) if c2 else 0):
                    lo, hi = max(a, p * self.page), min(a + c2, (p + 1) * self.page)
                    if p >= table.shape[1] or not 0 <= int(table[i, p]) < self.count:
                        continue
                    pid, part = int(table[i, p]), x[base + lo - a: base + hi - a].transpose(0, 1)
                    W, S = self.want_codes[which], self.want_scales[which]
                    keep = lo - p * self.page
                    for h in range(self.H):
                        new = part[h]
                        fin = torch.isfinite(new)
                        top = new[fin].abs().max().item() if fin.any() else 0.0
                        s = float(np.float32(top) / np.float32(127))
                        if keep:
                            s = max(s, S[pid, h].item())
                        if keep and s > S[pid, h].item():
                            W[pid, h, :keep] = (W[pid, h, :keep] * S[pid, h] / s).round()
                        q = (torch.where(fin, new, 0.0) / (s if s > 0 else 1.0)).round().clamp(-127, 127)
                        q = torch.where(new == math.inf, 127.0, torch.where(new == -math.inf, -127.0, q))
                        W[pid, h, keep: keep + hi - lo] = q
                        S[pid, h] = s
                base += c

    def check(self):
        for which in range(2):
            assert torch.equal(self.scales[which].double().cpu(), self.want_scales[which])
            assert torch.equal(self.codes[which].double().cpu(), self.want_codes[which])

    def read(self, lens, starts, dt, most=None):
        cu, st = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist()), _i32(starts)
        out = [torch.full((sum(lens) + 2, self.H * self.D + 8), 9.0, dtype=dt, device="cuda") for _ in range(2)]
        self.ops.cache_read(self.handle, _code(self.ops, dt), out[0].data_ptr(), out[0].stride(0), out[1].data_ptr(),
                            out[1].stride(0), cu.data_ptr(), st.data_ptr(), self.table.data_ptr(), self.table.shape[1],
                            self.n, max(lens) if most is None else most, stream=_stream())
        torch.cuda.synchronize()
        return out

    def rows(self, which, i, L):
        """Values of sequence i's first L positions, [L, H, D] in 64 bits, and which of them have a page."""
        at = torch.arange(L)
        per = self.table.shape[1]
        pid = self.table.cpu()[i][(at // self.page).clamp(max=per - 1)].long()
        ok = (at // self.page < per) & (pid >= 0) & (pid < self.count)
        pid = pid.clamp(0, self.count - 1)
        c, s = self.codes[which].cpu(), self.scales[which].double().cpu()
        return torch.where(ok[:, None, None], c[pid, :, at % self.page].double() * s[pid][:, :, None], 0.0), ok


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,D,page", [(1, 64, 16), (3, 64, 32), (2, 128, 16), (5, 128, 64), (16, 64, 64)])
def test_cache_write_codes_and_scales(ops, H, D, page, dt):
    """Codes and scales are equal to the definition's, bit for bit: first rows behind nothing, runs that
    end inside a page, single rows whose values outgrow the page's scale and shrink again."""
    n = 4
    c = Paged(ops, n, 300, H, D, page, 11)
    g = _gen(12)
    at = [0, 0, page - 1, 5]
    for step, lens in enumerate([[70, 1, 200, 17], [1, 1, 1, 1], [0, 2, 1, 33], [page, 0, 3, 1]]):
        T = sum(lens)
        size = [1.0, 3.0, 0.1, 10.0][step]
        k = (torch.randn(T, H * D, generator=g, device="cuda") * size).to(DT[dt])
        v = (torch.randn(T, H * D + 8, generator=g, device="cuda") * size).to(DT[dt])[:, : H * D]
        c.write(k, v, lens, at)
        c.check()
        at = [a + l for a, l in zip(at, lens)]
    dst = torch.bfloat16 if dt == "f16" else torch.float16  # read back in either type
    for out_dt in (DT[dt], dst):
        lens, starts = [a - min(a, 40) if i % 2 else a for i, a in enumerate(at)], [min(a, 40) if i % 2 else 0 for i, a in enumerate(at)]
        got = c.read(lens, starts, out_dt)
        for which in range(2):
            want = torch.cat([c.rows(which, i, s + l)[0][s:] for i, (l, s) in enumerate(zip(lens, starts))]).reshape(sum(lens), -1)
            have = got[which][: sum(lens), : H * D].double().cpu()
            # one product in fp32 and one rounding
            assert ((have - want).abs() <= (_u(out_dt) * (1 + 2.0 ** -10) + 2.0 ** -24) * want.abs() + torch.finfo(out_dt).tiny * _u(out_dt)).all()
            assert (got[which][sum(lens):] == 9).all() and (got[which][:, H * D:] == 9).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_cache_write_ties_and_odd_values(ops, dt):
    """Quotients at and next to a half, subnormal values, zeros, infinities and NaN."""
    H, D, page = 2, 64, 16
    c = Paged(ops, 1, 64, H, D, page, 21)
    k = torch.zeros(40, H, D, dtype=DT[dt], device="cuda")
    half = torch.arange(D, device="cuda").float() - 31.5  # scale 1: every value a tie
    k[0, 0] = half.to(DT[dt])
    k[1, 0, 0] = 127.0
    k[2, 0] = (torch.arange(D, device="cuda").float() * 0.5 + 0.5 * 2 ** -7).to(DT[dt])
    k[3, 1, 5] = float("inf")
    k[4, 1, 6] = -float("inf")
    k[5, 1, 7] = float("nan")
    k[6, 1, 8] = 2.5
    k[17, 0, 1] = torch.finfo(DT[dt]).smallest_normal / 4
    k[17, 0, 2] = -torch.finfo(DT[dt]).smallest_normal / 8
    k[18, 1, 3] = float("inf")  # nothing finite but zeros
    k[33] = torch.finfo(DT[dt]).max
    v = (torch.randn(40, H, D, generator=_gen(3), device="cuda") * 2.0 ** -20).to(DT[dt])
    c.write(k.view(40, -1), v.view(40, -1), [40], [0])
    c.check()


def test_cache_skips_bad_pages_and_bounds(ops):
    """Pages outside the cache, positions past the table, negative starts and rows past the bound are
    left out of writes and read back as 0; nothing else changes."""
    H, D, page = 2, 64, 16
    c = Paged(ops, 3, 96, H, D, page, 31)
    c.table[0, 1] = -1
    c.table[1, 2] = c.count
    c.table[2, 5] = 2 ** 31 - 1
    g = _gen(32)
    lens, starts = [60, 50, 40], [3, 0, 70]  # the last runs past its table of 96 positions
    k, v = [torch.randn(150, H * D, generator=g, device="cuda").half() for _ in range(2)]
    c.write(k, v, lens, starts)
    c.check()
    got = c.read([80, 70, 60], [0, 0, 60], torch.float16)
    base = 0
    for i, (l, s) in enumerate([(80, 0), (70, 0), (60, 60)]):
        want, ok = c.rows(0, i, s + l)
        have = got[0][base: base + l, : H * D].double().cpu().view(l, H, D)
        assert (have[~ok[s:]] == 0).all() and (~ok[s:]).any()
        assert ((have - want[s:]).abs() <= 1.01 * _u(torch.float16) * want[s:].abs() + 1e-7).all()
        base += l
    c.write(k, v, [20, 0, 9], [40, 7, 33], most=5)  # rows past the bound
    c.check()
    before = [x.clone() for x in c.codes + c.scales]
    cu, start = _i32([0, 5, 5, 5]), _i32([-2, 0, 0])
    ops.cache_write(c.handle, ops.DT_F16, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), cu.data_ptr(),
                    start.data_ptr(), c.table.data_ptr(), c.table.shape[1], 3, 5, stream=_stream())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, c.codes + c.scales))


# ---------------------------------------------------------------------------------------------
# attention over the cache


def _attention(ops, c, q, heads, lens, keys, scale, window=-1, most=None, max_kv=None, stream=None):
    T = sum(lens)
    out = torch.full((T + 1, heads * c.D + 8), 5.0, dtype=q.dtype, device="cuda")
    lse = torch.full((T + 1, heads), 5.0, device="cuda")
    cu, ln = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist()), _i32(keys)
    mq, mk = max(lens) if most is None else most, max(keys) if max_kv is None else max_kv
    ws = torch.empty(max(1, ops.cache_attention_workspace(c.handle, heads, c.n, mq, mk)), dtype=torch.uint8, device="cuda")
    ops.cache_attention(c.handle, _code(ops, q.dtype), q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads,
                        cu.data_ptr(), ln.data_ptr(), c.table.data_ptr(), c.table.shape[1], c.n, mq, mk, scale, window=window,
                        lse_ptr=lse.data_ptr(), workspace_ptr=ws.data_ptr(), workspace_bytes=ws.numel(),
                        stream=_stream() if stream is None else stream)
    torch.cuda.synchronize()
    return out, lse


def _check_attention(c, q, heads, lens, keys, scale, window, out, lse):
    """Bounds: a score is off by at most d = (D + 8) 2^-22 of the sum of its products' magnitudes (fp32
    sum; q's scaling and the key's scale are roundings within it), which moves its weight by the factor 1 + 2 d; a
    weight is rounded to 11 bits, summed over the keys, once; sums over L keys add L 2^-22; one rounding of the result.
    Weights (times their page's value scale) are f16 with the largest at 2^14 or above, whose smallest step is 2^-24: one far below
    the largest is off by up to 2^-39 of it, so each of the L keys adds 2^-39 of the largest weight times 128 at most."""
    G, base = heads // c.H, 0
    for i, (n, L) in enumerate(zip(lens, keys)):
        K, ok = c.rows(0, i, L)
        V, _ = c.rows(1, i, L)
        K, V, ok = K.cuda(), V.cuda(), ok.cuda()
        at = (torch.arange(L, device="cuda") // c.page).clamp(max=c.table.shape[1] - 1)
        vs = c.scales[1].double()[c.table[i].long().clamp(0, c.count - 1)[at]].nan_to_num(0.0)  # [L, H]
        x = q[base: base + n, : heads * c.D].double().view(n, heads, c.D)
        pos = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        seen = (j <= pos) & ok[None]
        if window >= 0:
            seen &= j >= pos - window
        for h in range(heads):
            s = (x[:, h] @ K[:, h // G].t() * scale).masked_fill(~seen, -math.inf)
            d = (c.D + 8) * 2.0 ** -22 * abs(scale) * ((x[:, h].abs() @ K[:, h // G].abs().t()).masked_fill(~seen, 0).amax(1) if L else x.new_zeros(n))
            none = ~seen.any(1)
            p = torch.softmax(s, 1).nan_to_num(0.0) if L else s
            want, mass = p @ V[:, h // G], p @ V[:, h // G].abs()
            have = out[base: base + n, h * c.D: (h + 1) * c.D].double()
            bound = _u(q.dtype) * want.abs() + mass * (2.0 ** -11 + 4 * d[:, None] + (L + 64) * 2.0 ** -22) + torch.finfo(q.dtype).tiny
            if L:
                bound += L * 2.0 ** -39 * 128 * (p * vs[:, h // G]).amax(1)[:, None]
            err = (have - want).abs()
            assert (err <= bound).all(), (i, h, (err / bound).max().item())
            assert (have[none] == 0).all() and (lse[base: base + n, h][none] == -math.inf).all()
            wl = torch.logsumexp(s, 1)[~none] if L else s.new_zeros(0)
            hl = lse[base: base + n, h][~none].double()
            assert ((hl - wl).abs() <= 2 * d[~none] + (L + 64) * 2.0 ** -22 + 2.0 ** -21 * (1 + wl.abs())).all()
        base += n
    assert (out[base:] == 5).all() and (out[:, heads * c.D:] == 5).all() and (lse[base:] == 5).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,G,D,page,lens,keys,window", [
    (1, 1, 64, 16, [1], [1], -1), (2, 1, 64, 16, [1], [17], -1), (1, 8, 128, 32, [1], [700], -1),
    (2, 4, 128, 16, [1, 1, 1, 1], [1, 15, 16, 1000], -1), (3, 5, 64, 64, [1, 1, 1], [63, 64, 65], -1),
    (2, 3, 64, 32, [1, 1, 1], [0, 300, 129], -1), (1, 16, 128, 64, [1, 1], [4000, 2], -1),
    (1, 40, 64, 16, [1, 2], [333, 20], -1), (2, 2, 128, 16, [5, 1, 3], [5, 40, 200], -1),
    (2, 1, 64, 64, [130, 17], [130, 400], -1), (1, 4, 128, 32, [64, 65, 1], [64, 1000, 77], -1),
    (2, 2, 64, 16, [3, 70, 1], [2, 100, 50], -1), (2, 2, 64, 16, [1, 40, 9], [900, 40, 300], 0),
    (1, 3, 128, 32, [1, 40, 100], [900, 500, 300], 64), (2, 1, 64, 16, [1, 33], [5000, 2100], 1000)])
def test_cache_attention(ops, H, G, D, page, lens, keys, window, dt):
    n, heads = len(lens), H * G
    c = Paged(ops, n, max(keys) + 1, H, D, page, 41)
    c.scales[1][::3] *= 30  # value scales that differ from page to page
    g = _gen(42)
    q = torch.randn(sum(lens), heads * D + 16, generator=g, device="cuda").to(DT[dt])
    scale = 1 / math.sqrt(D)
    out, lse = _attention(ops, c, q, heads, lens, keys, scale, window)
    _check_attention(c, q, heads, lens, keys, scale, window, out, lse)


def test_cache_attention_outside_pages_and_bounds(ops):
    """Keys on pages outside the cache are masked, a sequence of such pages alone has an empty row; what the
    unread rows hold (largest codes and scales) does not count; bounds wider than the batch do not matter."""
    H, D, page, heads = 2, 64, 16, 6
    c = Paged(ops, 4, 200, H, D, page, 51)
    c.table[0, 1] = -5
    c.table[0, 2] = c.count + 7
    c.table[1, :] = -1
    lens, keys = [2, 3, 1, 7], [100, 40, 23, 200]
    pid = int(c.table[2, 1])  # rows 7.. of this page lie behind the sequence's last
    c.codes[0][pid, :, 7:] = 127
    c.codes[1][pid, :, 7:] = -128
    for t in c.scales:  # pages that nobody reads
        used = set(c.table.cpu().flatten().tolist())
        for p in range(c.count):
            if p not in used:
                t[p] = float("nan")
    q = torch.randn(sum(lens), heads * D, generator=_gen(52), device="cuda").bfloat16()
    for most, max_kv in [(None, None), (20, 5000), (7, 200)]:
        out, lse = _attention(ops, c, q, heads, lens, keys, 0.125, most=most, max_kv=max_kv)
        _check_attention(c, q, heads, lens, keys, 0.125, -1, out, lse)


def test_cache_attention_past_its_table(ops):
    """Positions past the page table have no page: they are masked."""
    c = Paged(ops, 2, 64, 1, 64, 16, 53)
    q = torch.randn(3, 2 * 64, generator=_gen(54), device="cuda").half()
    lens, keys = [2, 1], [70, 120]
    out, lse = _attention(ops, c, q, 2, lens, keys, 0.125)
    _check_attention(c, q, 2, lens, keys, 0.125, -1, out, lse)


def test_cache_attention_replayed_with_other_lengths(ops):
    """A captured call over a cache long enough to be split (so two kernels), replayed with other lengths and
    tables, one of them an empty sequence."""
    H, D, page, heads = 2, 128, 32, 4
    c = Paged(ops, 2, 3000, H, D, page, 55)
    q = torch.randn(2, heads * D, generator=_gen(56), device="cuda").half()
    out = torch.full((3, heads * D + 8), 5.0, dtype=torch.float16, device="cuda")
    lse = torch.full((3, heads), 5.0, device="cuda")
    cu, ln = _i32([0, 1, 2]), _i32([3000, 17])
    ws = torch.empty(ops.cache_attention_workspace(c.handle, heads, 2, 1, 3000), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call():
        ops.cache_attention(c.handle, ops.DT_F16, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads,
                            cu.data_ptr(), ln.data_ptr(), c.table.data_ptr(), c.table.shape[1], 2, 1, 3000, 0.088,
                            lse_ptr=lse.data_ptr(), workspace_ptr=ws.data_ptr(), workspace_bytes=ws.numel(), stream=_stream())

    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for keys in ([3000, 17], [1, 2999], [0, 1500], [2048, 2049]):
        ln.copy_(_i32(keys))
        c.table.copy_(c.table.flip(0).clone())
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(c, q, heads, [1, 1], keys, 0.088, -1, out, lse)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("D,H,G,lens,keys,window", [
    (64, 2, 4, [40, 300, 7], [40, 1000, 700], -1), (128, 1, 8, [129, 16, 1], [500, 16, 3000], -1),
    (128, 2, 3, [200, 90, 64], [900, 2500, 64], 500), (64, 1, 33, [1, 1, 4], [5000, 0, 2], -1)])
def test_cache_attention_prompts(ops, D, H, G, lens, keys, window, page, dt):
    """Many query rows: tiles of 128 rows that end inside a sequence, windows, pages of every size, and a
    group so wide that one token's rows make a tile."""
    c = Paged(ops, 3, max(keys) + 1, H, D, page, 57)
    c.scales[1][::5] *= 20
    c.table[0, 2] = -1
    q = torch.randn(sum(lens), H * G * D, generator=_gen(58), device="cuda").to(DT[dt])
    scale = 1 / math.sqrt(D)
    out, lse = _attention(ops, c, q, H * G, lens, keys, scale, window)
    _check_attention(c, q, H * G, lens, keys, scale, window, out, lse)


@pytest.mark.parametrize("many", [0, 1])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_cache_attention_scores_and_scales_far_apart(ops, dt, many):
    """Scores in the hundreds that grow along the keys, queries from 2^-12 to 2^12, pages whose values are all zero
    (scale 0), value scales 2^16 apart."""
    H, D, page, heads = 2, 128, 16, 8
    c = Paged(ops, 3, 600, H, D, page, 61)
    per = c.table.shape[1]
    for i in range(3):
        for p in range(per):
            pid = int(c.table[i, p])
            c.scales[0][pid] *= 1 + 3 * p / per
            c.scales[1][pid] *= 2.0 ** (-8 + 16 * ((p * 7) % 5) / 4)
            if p % 9 == 4:
                c.scales[1][pid] = 0
                c.codes[1][pid] = 0
    lens, keys = [[1, 4, 1], [1, 30, 12]][many], [600, 555, 16 * 5]
    q = torch.randn(sum(lens), heads * D, generator=_gen(62), device="cuda")
    q = (q * torch.exp2(torch.linspace(-12, 5, q.shape[0], device="cuda"))[:, None]).to(DT[dt])
    q[:, D: 2 * D] *= 2.0 ** -9
    out, lse = _attention(ops, c, q, heads, lens, keys, 0.088)
    _check_attention(c, q, heads, lens, keys, 0.088, -1, out, lse)


def test_cache_attention_all_values_zero(ops):
    c = Paged(ops, 1, 64, 1, 64, 16, 63)
    c.codes[1].zero_()
    c.scales[1].zero_()
    q = torch.randn(1, 64, generator=_gen(64), device="cuda").half()
    out, lse = _attention(ops, c, q, 1, [1], [50], 0.125)
    _check_attention(c, q, 1, [1], [50], 0.125, -1, out, lse)


@pytest.mark.parametrize("D,H,G,rows,L", [(64, 32, 2, 4, 8000), (128, 32, 4, 3, 4000), (128, 2, 8, 20, 3000), (64, 40, 8, 1, 6000)])
def test_cache_attention_rows_do_not_depend_on_each_other(ops, D, H, G, rows, L):
    """A row and head's bits are the same whatever the other rows and heads of the call hold: queries of zeros, whose
    scores never grow along the keys, or large ones, whose scores do."""
    heads = H * G
    for seed in range(3):
        c = Paged(ops, 1, L, H, D, 16, 73 + seed)
        q = torch.randn(rows, heads, D, generator=_gen(74 + seed), device="cuda").half()
        keep = torch.zeros(rows, heads, dtype=torch.bool, device="cuda")
        keep.view(-1)[::3] = True
        got = []
        for by in (0, 8):
            x = torch.where(keep[..., None], q, q * by)
            out, lse = _attention(ops, c, x.view(rows, -1), heads, [rows], [L], 0.1)
            got.append((out[:rows, : heads * D].reshape(rows, heads, D), lse[:rows]))
        assert torch.equal(got[0][0][keep], got[1][0][keep]) and torch.equal(got[0][1][keep], got[1][1][keep])
        assert not torch.equal(got[0][0], got[1][0])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D,H,G,rows,L", [(64, 2, 3, 2, 100), (128, 2, 3, 2, 3000), (128, 1, 4, 3, 70001), (64, 1, 8, 30, 120),
                                          (128, 2, 8, 20, 3000)])
def test_cache_attention_queries_that_are_not_finite(ops, D, H, G, rows, L, dt):
    """A query with a NaN or infinity gives NaN, whether its keys are split between blocks (and joined) or not,
    for few rows and for many; every other row and head keeps its bits."""
    heads = H * G
    c = Paged(ops, 1, L, H, D, 16, 71)
    q = torch.randn(rows, heads * D, generator=_gen(72), device="cuda").to(DT[dt])
    clean, clean_lse = _attention(ops, c, q, heads, [rows], [L], 0.1)
    assert torch.isfinite(clean).all()
    q = q.view(rows, heads, D)
    bad = torch.zeros(rows, heads, dtype=torch.bool, device="cuda")
    for r, h, d, value in [(0, 1, 5, math.nan), (rows - 1, heads - 1, D - 1, math.nan), (rows // 2, 0, 0, math.inf),
                           (rows - 1, 0, 33, -math.inf)]:
        q[r, h, d], bad[r, h] = value, True
    out, lse = _attention(ops, c, q.view(rows, -1), heads, [rows], [L], 0.1)
    have = out[:rows, : heads * D].reshape(rows, heads, D)
    assert torch.isnan(have[bad]).all() and torch.isnan(lse[:rows][bad]).all()
    assert torch.equal(have[~bad], clean[:rows, : heads * D].reshape(rows, heads, D)[~bad])
    assert torch.equal(lse[:rows][~bad], clean_lse[:rows][~bad])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,G,D,lens,keys", [(2, 2, 64, [3, 2, 2], [2, 40, 60]), (1, 4, 128, [40, 33, 50], [30, 200, 90]),
                                             (1, 3, 64, [3, 2, 1], [2, 3000, 5])])
def test_cache_attention_queries_that_are_not_finite_and_see_no_key(ops, H, G, D, lens, keys, dt):
    """NaN and infinities in a query whose keys all lie on pages outside the cache, or which stands before the first
    position: 0 and -inf as for any query without a key."""
    heads = H * G
    c = Paged(ops, 3, max(keys), H, D, 16, 75)
    c.table[1] = -1
    q = torch.randn(sum(lens), heads * D, generator=_gen(76), device="cuda").to(DT[dt])
    q[0, 3], q[lens[0], 5], q[lens[0] + 1, 0] = math.nan, math.nan, -math.inf
    out, lse = _attention(ops, c, q, heads, lens, keys, 0.1)
    for rows in (slice(0, lens[0] - keys[0]), slice(lens[0], lens[0] + lens[1])):
        assert (out[rows, : heads * D] == 0).all() and (lse[rows] == -math.inf).all()
    seen = torch.cat([out[lens[0] - keys[0]: lens[0]], out[lens[0] + lens[1]: sum(lens)]])[:, : heads * D]
    assert torch.isfinite(seen).all() and seen.any()


@pytest.mark.parametrize("H,G,D,page,n,L", [(8, 2, 128, 64, 2, 70001), (1, 1, 64, 16, 1, 131072), (4, 16, 128, 32, 40, 20000)])
def test_cache_attention_long_caches_add_up(ops, H, G, D, page, n, L):
    """Long caches with a bound that stays far below the result. A warp's sums over its share of a chunk (at most 4096
    keys) take one step a key, each off by at most 2^-23 of what is summed; the four warps and then the chunks add
    one each. Scores and weights as in _check_attention."""
    c = Paged(ops, 1, L, H, D, page, 83)
    heads = H * G
    q = torch.randn(n, heads * D, generator=_gen(84), device="cuda").half() * 1.5
    scale = 1 / math.sqrt(D)
    out, lse = _attention(ops, c, q, heads, [n], [L], scale)
    steps = 4096 + 4 + -(-L // 128)
    K, V = [c.rows(which, 0, L)[0].cuda() for which in (0, 1)]
    x = q.double().view(n, heads, D)
    pos = torch.arange(L - n, L, device="cuda")[:, None]
    hidden = torch.arange(L, device="cuda")[None] > pos
    vs = c.scales[1].max().item()
    larger = []
    for h in range(heads):
        s = (x[:, h] @ K[:, h // G].t() * scale).masked_fill(hidden, -math.inf)
        d = (D + 8) * 2.0 ** -22 * scale * (x[:, h].abs() @ K[:, h // G].abs().t()).amax(1)
        p = torch.softmax(s, 1)
        want, mass = p @ V[:, h // G], p @ V[:, h // G].abs()
        bound = _u(q.dtype) * want.abs() + mass * (2.0 ** -11 + 2 * d[:, None] + 2 * steps * 2.0 ** -23) + L * 2.0 ** -39 * 128 * vs * p.amax(1)[:, None]
        err = (out[:n, h * D: (h + 1) * D].double() - want).abs()
        assert (err <= bound).all(), (h, (err / bound).max().item())
        assert ((lse[:n, h].double() - torch.logsumexp(s, 1)).abs() <= d + steps * 2.0 ** -23 + 2.0 ** -22 * (1 + torch.logsumexp(s, 1).abs())).all()
        larger.append((bound < 0.5 * want.abs()).double().mean().item())
    assert np.mean(larger) > 0.75, np.mean(larger)  # so that a wrong result fails


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,G,D,n,L", [(4, 8, 128, 1, 20000), (2, 4, 64, 3, 300), (2, 4, 128, 40, 6000), (1, 1, 64, 100, 128)])
def test_cache_attention_results_are_as_near_as_their_type_allows(ops, H, G, D, n, L, dt):
    """The root mean square of the error against 64 bits is that of rounding the exact result, and a twentieth at most:
    rounding to bf16 leaves about 1.7e-3 of the results' size and to f16 2.1e-4; before it stand 2.4e-4 for bf16 alone
    (weights of 11 bits) and some 1e-5 (scores, sums)."""
    c = Paged(ops, 1, L, H, D, 32, 85)
    heads = H * G
    q = (torch.randn(n, heads * D, generator=_gen(86), device="cuda") * 0.5).to(DT[dt])
    out, _ = _attention(ops, c, q, heads, [n], [L], 0.1)
    K, V = [c.rows(which, 0, L)[0].cuda() for which in (0, 1)]
    hidden = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
    x = q.double().view(n, heads, D)
    want = torch.cat([torch.softmax((x[:, h] @ K[:, h // G].t() * 0.1).masked_fill(hidden, -math.inf), 1) @ V[:, h // G]
                      for h in range(heads)], 1)
    rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
    least = rms(want.to(DT[dt]).double() - want)
    assert rms(out[:n, : heads * D].double() - want) <= 1.05 * least


FAR = [(64, 2, 4, [1, 2, 1], [100, 90, 300]), (128, 1, 4, [2], [3000]), (64, 1, 8, [30, 5, 50], [120, 90, 50]), (128, 2, 3, [40], [2500])]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D,H,G,lens,keys", FAR)
def test_cache_attention_far_larger_values_without_weight(ops, D, H, G, lens, keys, dt):
    """Pages with values up to the end of fp32 (what padding of any bits may leave), at keys whose weights are far below
    its smallest number or that a row does not see, change nothing; rows in one block with them and rows whose keys
    are split."""
    n, heads = len(lens), H * G
    c = Paged(ops, n, max(keys), H, D, 16, 87)
    last = [int(c.table[i, (L - 1) // 16]) for i, L in enumerate(keys)]  # hidden from the rows before it
    for p in c.table[:, 2::5].flatten().tolist() + last:
        c.codes[0][p], c.codes[1][p] = -127, 127
        c.scales[0][p], c.scales[1][p] = 1.0, 3e38
    q = (torch.rand(sum(lens), heads * D, generator=_gen(88), device="cuda") + 0.5).to(DT[dt])
    out, lse = _attention(ops, c, q, heads, lens, keys, 0.3)
    _check_attention(c, q, heads, lens, keys, 0.3, -1, out, lse)
    assert out[: sum(lens), : heads * D].abs().max() < 10


@pytest.mark.parametrize("D,H,G,lens,keys", FAR)
def test_cache_attention_value_scales_over_the_whole_range(ops, D, H, G, lens, keys):
    """Value scales from 2^-120 to 2^100, with zero scales (and zero codes) among them; half of the sequences' pages
    lie within a narrower range, so that some blocks take the common way."""
    n, heads = len(lens), H * G
    c = Paged(ops, n, max(keys), H, D, 16, 89)
    g = _gen(90)
    c.scales[1] = torch.exp2(torch.rand(c.count, H, generator=g, device="cuda") * 220 - 120)
    c.scales[1][::7], c.codes[1][::7] = 0, 0
    if n > 1:
        c.scales[1][c.table[1].long()] = torch.exp2(torch.rand(c.table.shape[1], H, generator=g, device="cuda") * 80)
    c.handle = ops.Cache(c.codes[0].data_ptr(), c.codes[1].data_ptr(), c.scales[0].data_ptr(), c.scales[1].data_ptr(), c.count, 16, H, D)
    q = torch.randn(sum(lens), heads * D, generator=g, device="cuda").bfloat16()
    q[::2] *= 8  # weights far apart too
    out, lse = _attention(ops, c, q, heads, lens, keys, 0.1)
    _check_attention(c, q, heads, lens, keys, 0.1, -1, out, lse)


@pytest.mark.parametrize("lens,keys", [([2, 0, 1, 0, 3], [300, 200, 90, 0, 64]), ([0, 40, 0, 5, 90], [7, 300, 2, 90, 90])])
def test_cache_attention_sequences_without_queries_and_shared_pages(ops, lens, keys):
    """Sequences with no query row between others, pages that several sequences name (a common beginning) and pages
    that one table row names twice."""
    c = Paged(ops, 5, 320, 2, 64, 16, 91)
    c.table[1:, :3] = c.table[0, :3]
    c.table[0, 4], c.table[2, 5] = c.table[0, 1], c.table[2, 3]
    q = torch.randn(sum(lens), 6 * 64, generator=_gen(92), device="cuda").bfloat16()
    out, lse = _attention(ops, c, q, 6, lens, keys, 0.125)
    some = [i for i, n in enumerate(lens) if n]
    c.table, c.n = c.table[some].contiguous(), len(some)
    _check_attention(c, q, 6, [lens[i] for i in some], [keys[i] for i in some], 0.125, -1, out, lse)


def test_cache_calls_with_rows_far_apart(ops):
    """Row strides that take offsets past 2^31 elements, in every call on a cache."""
    H, D, n, stride = 2, 64, 3, 2 ** 30 + 8
    if torch.cuda.mem_get_info()[0] < 60 * 2 ** 30:
        pytest.skip("needs 60 GB")
    c = Paged(ops, 1, 40, H, D, 16, 93)
    big = [torch.empty(2 * stride + 4 * H * D, dtype=torch.float16, device="cuda") for _ in range(4)]
    k, v, q, out = [x.as_strided((n, H * D), (stride, 1)) for x in big]
    for i, x in enumerate((k, v, q)):
        x.copy_(torch.randn(n, H * D, generator=_gen(94 + i), device="cuda"))
    c.write(k, v, [n], [20])
    c.check()
    lse, cu, ln = torch.empty(n, H, device="cuda"), _i32([0, n]), _i32([20 + n])
    ops.cache_attention(c.handle, ops.DT_F16, q.data_ptr(), stride, out.data_ptr(), stride, H, cu.data_ptr(), ln.data_ptr(),
                        c.table.data_ptr(), c.table.shape[1], 1, n, 20 + n, 0.125, lse_ptr=lse.data_ptr(), stream=_stream())
    want, want_lse = _attention(ops, c, q.contiguous(), H, [n], [20 + n], 0.125)
    assert torch.equal(out, want[:n, : H * D]) and torch.equal(lse, want_lse[:n])
    ops.cache_read(c.handle, ops.DT_F16, k.data_ptr(), stride, v.data_ptr(), stride, cu.data_ptr(), _i32([20]).data_ptr(),
                   c.table.data_ptr(), c.table.shape[1], 1, n, stream=_stream())
    near = c.read([n], [20], torch.float16)
    assert torch.equal(k, near[0][:n, : H * D]) and torch.equal(v, near[1][:n, : H * D])


def test_cache_attention_one_workspace_for_smaller_calls(ops):
    """One buffer of the largest batch's size, with known bytes behind it, through calls that shrink in every
    direction and split their keys more than the largest does."""
    H, G, D, L = 2, 4, 64, 3000
    c = Paged(ops, 40, L, H, D, 16, 79)
    size = ops.cache_attention_workspace(c.handle, H * G, 40, 20, L)
    ws = torch.full((size + 64,), 7, dtype=torch.uint8, device="cuda")
    split = 0
    for n, rows, keys in [(40, 1, 2000), (9, 1, L), (1, 1, L), (1, 1, 200), (2, 20, L), (1, 9, 700), (40, 2, 150), (1, 1, 64)]:
        lens, at = [rows] * n, [max(rows, keys - 3 * i) for i in range(n)]
        q = torch.randn(n * rows, H * G * D, generator=_gen(80), device="cuda").bfloat16()
        out = torch.full((n * rows + 1, H * G * D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((n * rows + 1, H * G), 5.0, device="cuda")
        cu, ln = _i32([i * rows for i in range(n + 1)]), _i32(at)
        ws[:size] = 7
        ops.cache_attention(c.handle, ops.DT_BF16, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), H * G, cu.data_ptr(),
                            ln.data_ptr(), c.table.data_ptr(), c.table.shape[1], n, rows, keys, 0.125, lse_ptr=lse.data_ptr(),
                            workspace_ptr=ws.data_ptr(), workspace_bytes=size, stream=_stream())
        torch.cuda.synchronize()
        assert (ws[size:] == 7).all()
        split += int((ws[:size] != 7).any())
        _check_attention(c, q, H * G, lens, at, 0.125, -1, out, lse)
    assert 2 <= split < 8


def test_cache_attention_waits_that_run_out_give_nan(ops):
    """A tile of keys that never comes (short waits, the library's own self-test): the rows are NaN, split keys or not,
    few rows or many, and the kernels end; calls behind it are as ever."""
    import time
    from sys1rust_b200 import backend
    t = time.perf_counter()
    assert backend.selftest_cache_attention_timeout(0, 10_000_000) == [1, 1, 1, 1]
    assert time.perf_counter() - t < 5
    c = Paged(ops, 1, 300, 2, 64, 16, 77)
    q = torch.randn(2, 4 * 64, generator=_gen(78), device="cuda").half()
    out, lse = _attention(ops, c, q, 4, [2], [300], 0.1)
    _check_attention(c, q, 4, [2], [300], 0.1, -1, out, lse)


def test_cache_attention_long_cache(ops):
    """70001 positions, more than 2^31 bytes into the codes' array for the last pages."""
    H, D, page, L = 8, 128, 64, 70001
    per = -(-L // page)
    big = 2 ** 31 // (H * page * D) + 64  # pages before the sequence's own
    free, _ = torch.cuda.mem_get_info()
    if free < 8 * 2 ** 30:
        pytest.skip("needs 8 GB")
    g = _gen(71)
    codes = [torch.zeros(big + per, H, page, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    for x in codes:
        x[big:] = torch.randint(-127, 128, (per, H, page, D), generator=g, device="cuda", dtype=torch.int8)
    scales = [torch.rand(big + per, H, generator=g, device="cuda") * 0.02 for _ in range(2)]
    table = (big + torch.randperm(per, generator=g, device="cuda")).to(torch.int32)[None].contiguous()
    handle = ops.Cache(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), big + per, page, H, D)
    c = Paged.__new__(Paged)
    c.H, c.D, c.page, c.n, c.ops, c.count, c.table, c.handle = H, D, page, 1, ops, per, table, handle
    q = torch.randn(2, H * 2 * D, generator=g, device="cuda").bfloat16()
    out, lse = _attention(ops, c, q, 2 * H, [2], [L], 0.088)
    c.table = table - big
    c.codes, c.scales = [x[big:] for x in codes], [x[big:] for x in scales]
    _check_attention(c, q, 2 * H, [2], [L], 0.088, -1, out, lse)


# ---------------------------------------------------------------------------------------------
# sampling


def _sample_ref(x, u, T, k, p, m):
    """(token, probability, how near u or p comes to another outcome) of one row, in 64 bits."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or x.max() == -np.inf:
        return -1, 0.0, 1.0
    if not T > 0:
        return int(x.argmax()), 1.0, 1.0
    e = np.exp((x - x.max()) / T)
    order = np.lexsort((np.arange(x.size), -x))
    if k > 0:
        order = order[:k]
    near = 1.0
    if p < 1:
        cum = np.cumsum(e[order])
        cut = int(np.searchsorted(cum, p * cum[-1], side="left")) + 1 if p > 0 else 1
        near = min(near, np.abs(cum / cum[-1] - p).min())
        order = order[:cut]
    if m > 0:
        near = min(near, np.abs(e[order] / min(m, 1.0) - 1)[1:].min(initial=1.0))
        order = order[e[order] >= min(m, 1.0)]
    order = np.sort(order)
    cum = np.cumsum(e[order])
    order, cum = order[cum > 0], cum[cum > 0]
    j = min(int(np.searchsorted(cum, u * cum[-1], side="right")), int(np.flatnonzero(e[order])[-1])) if u == u else int(np.flatnonzero(e[order])[-1])
    if u == u:
        near = min(near, np.abs(cum[:-1] / cum[-1] - u).min(initial=1.0)) if 0 < u < 1 else near
    return int(order[j]), float(e[order[j]] / cum[-1]), near


def _sample(ops, x, u, T=None, k=None, p=None, m=None, prob=True):
    R, V = x.shape
    token = torch.full((R + 1,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((R + 1,), -7.0, device="cuda") if prob else None
    ops.sample(_code(ops, x.dtype), x.data_ptr(), x.stride(0), R, V, token.data_ptr(), u.data_ptr(), temperature_ptr=_ptr(T),
               top_k_ptr=_ptr(k), top_p_ptr=_ptr(p), min_p_ptr=_ptr(m), prob_ptr=_ptr(pr), stream=_stream())
    torch.cuda.synchronize()
    assert token[R] == -7 and (pr is None or pr[R] == -7)
    return token[:R].cpu().numpy(), None if pr is None else pr[:R].cpu().numpy()


def _check_sample(ops, x, u, T, k, p, m):
    token, prob = _sample(ops, x, u, T, k, p, m)
    xs = x.float().cpu().numpy()
    R = x.shape[0]
    get = lambda t, d: np.full(R, d) if t is None else t.cpu().numpy()  # noqa: E731
    Ts, ks, ps, ms, us = get(T, 1.0), get(k, 0), get(p, 1.0), get(m, 0.0), u.cpu().numpy()
    decided = 0
    for r in range(R):
        want, pw, near = _sample_ref(xs[r], float(us[r]), float(Ts[r]), int(ks[r]), float(ps[r]), float(ms[r]))
        # masses carry 3e-8 each; a border nearer than 3e-7 is undecided
        if near > 3e-7:
            assert token[r] == want, (r, token[r], want, near)
            # the mass kept, summed, and the rounding of the share
            assert abs(prob[r] - pw) <= 3e-7 * pw + 1e-12, (r, prob[r], pw)
            decided += 1
        else:
            assert 0 <= token[r] < x.shape[1]
    # a row of V borders is undecided with a chance of at most 2 * 3e-7 * V: 8 % at the largest V here
    assert decided >= R / 2 or R < 10


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 1000, 1024, 1025, 50368, 131075])
def test_sample(ops, V, dt):
    """Rows with every combination of the filters, among them ones that keep a single token and ones that
    keep all; 16-bit logits bring many equal ones, so the order of equals decides."""
    R = 24
    g = _gen(81 + V)
    x = (torch.randn(R, V + 3, generator=g, device="cuda") * 2.5).to(DT[dt])[:, :V]
    u = torch.rand(R, generator=g, device="cuda")
    r = torch.arange(R, device="cuda")
    T = torch.where(r % 5 == 4, 0.05, 0.3 + 0.1 * (r % 12))
    k = torch.where(r % 2 == 0, 0, 1 + (r * r * 37) % max(V, 2)).to(torch.int32)
    p = torch.where(r % 3 == 0, 1.0, 0.04 * r)
    m = torch.where(r % 4 < 2, 0.0, 0.01 * r)
    _check_sample(ops, x, u, T, k, p, m)
    _check_sample(ops, x, u, None, None, None, None)
    _check_sample(ops, x, u, T, k, None, None)
    _check_sample(ops, x, u, T, None, p, None)
    _check_sample(ops, x, u, None, None, None, m)
    token, _ = _sample(ops, x, u, T, k, p, m, prob=False)
    assert (token == _sample(ops, x, u, T, k, p, m)[0]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_sample_equal_and_masked_logits(ops, dt):
    """All logits equal (in one bin of every histogram), two values, -inf in most places, one finite logit
    alone, zeros of both signs, temperatures from tiny to huge."""
    V, R = 5000, 40
    g = _gen(91)
    x = torch.zeros(R, V, dtype=DT[dt], device="cuda")
    x[8:16] = torch.where(torch.rand(8, V, generator=g, device="cuda") < 0.5, 1.0, -1.0).to(DT[dt])
    x[16:24] = torch.where(torch.rand(8, V, generator=g, device="cuda") < 0.98, -math.inf, 3.0).to(DT[dt])
    x[24:32] = -math.inf
    x[24:32, 4321] = -5
    x[32:40, ::2] = -0.0
    x[0:4] = 60000.0
    u = torch.rand(R, generator=g, device="cuda")
    r = torch.arange(R, device="cuda")
    T = torch.tensor([1e-6, 0.7, 1.0, 1e6], device="cuda").repeat(10)
    k = torch.where(r % 8 < 4, 0, 1 + r * 13).to(torch.int32)
    p = torch.where(r % 3 == 1, 0.37, 1.0)
    _check_sample(ops, x, u, T, k, p, None)
    _check_sample(ops, x, u, None, k, None, torch.full((R,), 0.5, device="cuda"))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_sample_rows_without_a_distribution_and_odd_parameters(ops, dt):
    V = 700
    g = _gen(95)
    x = torch.randn(16, V, generator=g, device="cuda").to(DT[dt])
    x[0, 5] = math.nan
    x[1, 699] = math.inf
    x[2] = -math.inf
    x[3, 100:] = -math.inf
    x[4, 17] = x[4, 600] = 9
    u = torch.rand(16, generator=g, device="cuda")
    u[5], u[6], u[7], u[8] = 1.0, math.nan, 0.0, 2.0
    T = torch.ones(16, device="cuda")
    T[4], T[9], T[10] = 0.0, -1.0, math.nan
    T[0], T[11] = 0.0, math.inf
    k = torch.zeros(16, dtype=torch.int32, device="cuda")
    k[3], k[12], k[13] = 300, -4, 2 ** 31 - 1
    p = torch.ones(16, device="cuda")
    p[12], p[13], p[14] = 0.0, -1.0, math.nan
    m = torch.zeros(16, device="cuda")
    m[14], m[15] = math.nan, 7.0
    xs, us = x.float().cpu().numpy(), u.cpu().numpy()
    token, prob = _sample(ops, x, u, T, k, p, m)
    assert list(token[:3]) == [-1, -1, -1] and (prob[:3] == 0).all()
    assert token[4] == 17 and prob[4] == 1
    for r in (9, 10):
        assert token[r] == xs[r].argmax() and prob[r] == 1
    assert token[11] == min(V - 1, int(us[11] * V)) or abs(us[11] * V - round(us[11] * V)) < 1e-3
    assert token[12] == xs[12].argmax() and token[13] == xs[13].argmax() and token[15] == xs[15].argmax()
    for r in (3, 5, 6, 7, 8, 14):
        want, pw, near = _sample_ref(xs[r], float(us[r]), 1.0, int(k[r]), 1.0, 0.0)
        assert near < 3e-7 or (token[r] == want and abs(prob[r] - pw) <= 3e-7 * pw), r


@pytest.mark.parametrize("V", [5, 700, 50368])
def test_sample_infinite_temperature_with_filters(ops, V):
    """At T = inf every finite logit has e = 1: min-p keeps all of them, up to its largest value of 1; top-k and top-p
    keep the first ones in the order of the logits. 1 and above is one value of min-p at any temperature."""
    R = 12
    x = torch.randn(R, V, generator=_gen(98), device="cuda")
    x[:, 1] = -math.inf
    u = torch.rand(R, generator=_gen(99), device="cuda")
    T = torch.full((R,), math.inf, device="cuda")
    m = torch.tensor([0.0, 0.3, 1.0, 7.0, math.inf, 1e-38] * 2, device="cuda")
    k = torch.where(torch.arange(R, device="cuda") < 6, 0, 3).to(torch.int32)
    p = torch.where(torch.arange(R, device="cuda") % 2 == 0, 1.0, 0.49)
    for top_p in (None, p):
        token, prob = _sample(ops, x, u, T, k, top_p, m)
        for r in range(R):
            row = x[r].cpu().numpy()
            order = np.lexsort((np.arange(V), -row))[: V - 1]
            order = order[: 3] if k[r] else order
            if top_p is not None and p[r] < 1:  # those before which less than p of the mass lies
                order = order[: int(np.ceil(float(p[r]) * order.size))]
            order = np.sort(order)
            at = float(u[r]) * order.size
            assert abs(at - round(at)) < 1e-3 or token[r] == order[int(at)], (r, token[r])
            assert abs(prob[r] * order.size - 1) < 1e-6
    token, prob = _sample(ops, x, u, None, None, None, torch.full((R,), 3.0, device="cuda"))
    assert (token == x.argmax(1).cpu().numpy()).all() and (prob == 1).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,size", [(0.0, 2.5), (0.2, 0.5)])
def test_sample_rows_do_not_depend_on_their_batch(ops, dt, m, size):
    """The same row with the same numbers gives the same token and the same bits of its share alone (shared by eight
    blocks) and in a batch (one block a row), with values of top-p right at a border between two tokens."""
    V, R = 50368, 160
    x = (torch.randn(1, V, generator=_gen(96), device="cuda") * size).to(DT[dt])
    cum = np.cumsum(np.exp(np.sort(x[0].double().cpu().numpy())[::-1] - x.double().max().item()))
    p = torch.from_numpy((cum / cum[-1])[np.linspace(1, 3000, R).astype(int)].astype(np.float32)).cuda()
    u, mp = torch.full((R,), 0.9999, device="cuda"), torch.full((R,), m, device="cuda")
    token, prob = _sample(ops, x.expand(R, V).contiguous(), u, None, None, p, mp)
    alone = [_sample(ops, x, u[r: r + 1], None, None, p[r: r + 1], mp[r: r + 1]) for r in range(R)]
    assert token.tolist() == [int(t[0]) for t, _ in alone]
    assert prob.tolist() == [float(q[0]) for _, q in alone]
    assert len(set(prob.tolist())) > R / 2


def test_sample_rows_far_apart_and_the_largest_vocabulary(ops):
    """Rows whose offsets pass 2^31 elements; 2^18 logits, many equal, whose masses and counts fill their sums."""
    V, stride = 2 ** 18, 2 ** 31 + 2 ** 18
    if torch.cuda.mem_get_info()[0] < 20 * 2 ** 30:
        pytest.skip("needs 20 GB")
    x = torch.empty(stride + V, dtype=torch.bfloat16, device="cuda").as_strided((2, V), (stride, 1))
    g = _gen(94)
    for size in (0.0, 0.01, 3.0):
        x.copy_(torch.randn(2, V, generator=g, device="cuda") * size)
        u = torch.rand(2, generator=g, device="cuda")
        for k, p in [(None, None), (_i32([200000, 100]), None), (None, torch.tensor([0.9, 0.3], device="cuda")),
                     (_i32([50000, 0]), torch.tensor([0.77, 1.0], device="cuda"))]:
            _check_sample(ops, x, u, None, k, p, None)


def test_sample_values_over_the_whole_range(ops):
    """Logits from the smallest to the largest floats: a cut far below the largest, in one bin with others."""
    V, R = 3000, 8
    g = _gen(97)
    x = torch.randn(R, V, generator=g, device="cuda") * torch.exp2(torch.randint(-100, 100, (R, V), generator=g, device="cuda").float())
    x[4:] = torch.randn(4, V, generator=g, device="cuda") * 1e-6  # all in the first bins
    u = torch.rand(R, generator=g, device="cuda")
    k = _i32([5, 2000, 3000, 100, 5, 1700, 0, 29])
    p = torch.tensor([1, 0.5, 0.9, 1, 0.3, 0.77, 0.999, 0.01], device="cuda")
    for T in (1.0, 1e-6, 1e30):
        _check_sample(ops, x, u, torch.full((R,), T, device="cuda"), k, p, None)


# ---------------------------------------------------------------------------------------------
# together, on streams and in graphs


class Step:
    """A small layer and head: q, k, v from 4-bit products, appended, attended to, and a token sampled
    from 4-bit logits. Buffers are kept, lengths live on the GPU, so a captured step replays."""

    def __init__(self, ops, n=3, seed=7):
        self.ops, self.n = ops, n
        self.H, self.G, self.D, self.V = 2, 3, 64, 997
        H, G, D, V, width = self.H, self.G, self.D, self.V, 256
        g = _gen(seed)
        dt = torch.bfloat16
        sizes = {"qkv": (H * (G + 2) * D, width), "logits": (V, H * G * D)}
        self.w = {}
        for name, (N, K) in sizes.items():
            w = torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K) * 2
            codes, scales = ops.nibble_pack(w.cpu().numpy(), 32)
            self.w[name] = (torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda().to(dt))
        self.emb = torch.randn(V, width, generator=g, device="cuda").to(dt)
        self.x = torch.empty(n, width, dtype=dt, device="cuda")
        self.qkv = torch.empty(n, sizes["qkv"][0], dtype=dt, device="cuda")
        self.att = torch.empty(n, H * G * D, dtype=dt, device="cuda")
        self.logits = torch.empty(n, V, device="cuda")
        self.token = torch.arange(n, dtype=torch.int32, device="cuda")
        self.u = torch.empty(n, device="cuda")
        self.cache = Paged(ops, n, 40, H, D, 16, seed)
        self.cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        self.len = _i32([0, 5, 20][:n])
        self.ws = torch.empty(max(1, ops.cache_attention_workspace(self.cache.handle, H * G, n, 1, 40)), dtype=torch.uint8, device="cuda")
        self.p, self.T = torch.full((n,), 0.9, device="cuda"), torch.full((n,), 0.8, device="cuda")
        self.start = torch.empty_like(self.len)

    def run(self):
        ops, H, G, D, c, st = self.ops, self.H, self.G, self.D, self.cache, _stream()
        self.x.copy_(self.emb[self.token.long()])
        _nibble(ops, self.x, *self.w["qkv"], None, self.qkv, 256, 32)
        k, v = self.qkv[:, H * G * D:], self.qkv[:, H * (G + 1) * D:]
        self.start.copy_(self.len)
        ops.cache_write(c.handle, ops.DT_BF16, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), self.cu.data_ptr(),
                        self.start.data_ptr(), c.table.data_ptr(), c.table.shape[1], self.n, 1, stream=st)
        self.len.add_(1)
        ops.cache_attention(c.handle, ops.DT_BF16, self.qkv.data_ptr(), self.qkv.stride(0), self.att.data_ptr(),
                            self.att.stride(0), H * G, self.cu.data_ptr(), self.len.data_ptr(), c.table.data_ptr(),
                            c.table.shape[1], self.n, 1, 40, 0.125, workspace_ptr=self.ws.data_ptr(),
                            workspace_bytes=self.ws.numel(), stream=st)
        _nibble(ops, self.att, *self.w["logits"], None, self.logits, H * G * D, 32)
        ops.sample(ops.DT_F32, self.logits.data_ptr(), self.logits.stride(0), self.n, self.V, self.token.data_ptr(),
                   self.u.data_ptr(), temperature_ptr=self.T.data_ptr(), top_p_ptr=self.p.data_ptr(), stream=st)

    def check(self):
        """The step that has just run, part by part, each from the inputs it was given."""
        H, G, D, c = self.H, self.G, self.D, self.cache
        for x, (codes, scales), out, K in [(self.x, self.w["qkv"], self.qkv, 256), (self.att, self.w["logits"], self.logits, H * G * D)]:
            w = _nibble_weights(codes, scales, None, K, 32)
            ref = x.double() @ w.t()
            mag = x.double().abs() @ (scales.double()[:, torch.arange(K, device="cuda") // 32] * 30).t()
            assert ((out.double() - ref).abs() <= _u(out.dtype) * ref.abs() + (K + 64) * 2.0 ** -22 * mag).all()
        for i in range(self.n):
            L = int(self.len[i])
            for which, first in ((0, H * G * D), (1, H * (G + 1) * D)):
                row = self.qkv[i, first: first + H * D].double().view(H, D).cpu()
                have = c.rows(which, i, L)[0][-1]
                s = c.scales[which].double().cpu()[int(c.table[i, (L - 1) // 16])]
                assert ((have - row).abs() <= 0.5 * s[:, None] * (1 + 1e-6)).all()
        out = torch.full((self.n + 1, H * G * D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
        out[: self.n, : H * G * D] = self.att
        lse = torch.full((self.n + 1, H * G), 5.0, device="cuda")
        lens = [1] * self.n
        o2, lse2 = _attention(self.ops, c, self.qkv, H * G, lens, self.len.tolist(), 0.125)
        _check_attention(c, self.qkv, H * G, lens, self.len.tolist(), 0.125, -1, o2, lse2)
        del lse
        ref = o2[: self.n, : H * G * D].double()
        assert ((self.att.double() - ref).abs() <= 2.0 ** -7 * ref.abs() + 1e-4).all()
        for i in range(self.n):
            want, _, near = _sample_ref(self.logits[i].cpu().numpy(), float(self.u[i]), float(np.float32(0.8)), 0, float(np.float32(0.9)), 0.0)
            assert near < 3e-7 or int(self.token[i]) == want


def test_token_steps_eager_and_replayed(ops):
    """Steps one after another: eagerly, then the same from a captured graph on a side stream, bit for bit the same."""
    tokens = []
    for graph in (False, True):
        s = Step(ops)
        u = torch.rand(12, s.n, generator=_gen(8), device="cuda")
        run = s.run
        if graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            state = [t.clone() for t in (s.token, s.len, *s.cache.codes, *s.cache.scales)]
            with torch.cuda.stream(side):
                s.u.copy_(u[0])
                s.run()  # outside the capture first, as programs do
                side.synchronize()
                for t, old in zip((s.token, s.len, *s.cache.codes, *s.cache.scales), state):
                    t.copy_(old)
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr, stream=side):
                    s.run()
            torch.cuda.synchronize()
            run = gr.replay
        for i in range(12):
            s.u.copy_(u[i])
            run()
            torch.cuda.synchronize()
            if not graph and i % 5 == 0:
                s.check()
            tokens.append((graph, s.token.tolist(), s.logits.clone()))
    half = len(tokens) // 2
    for a, b in zip(tokens[:half], tokens[half:]):
        assert a[1] == b[1] and torch.equal(a[2], b[2])


def test_two_streams_at_once(ops):
    """Two sequences of steps on two streams, nothing waiting between them, each as if alone."""
    alone = []
    for seed in (1, 2):
        s = Step(ops, seed=seed)
        s.u.fill_(0.4)
        for _ in range(10):
            s.run()
        torch.cuda.synchronize()
        alone.append((s.token.clone(), s.logits.clone()))
    steps = [Step(ops, seed=seed) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in steps]
    for s in steps:
        s.u.fill_(0.4)
    torch.cuda.synchronize()
    for _ in range(10):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.run()
    torch.cuda.synchronize()
    for s, (token, logits) in zip(steps, alone):
        assert torch.equal(s.token, token) and torch.equal(s.logits, logits)


def test_host_memory_is_refused(ops):
    from sys1rust_b200.backend import BackendError
    x = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
    codes = torch.zeros(8, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(8, 2, dtype=torch.float16, device="cuda")
    out = torch.zeros(1, 8, dtype=torch.float16)
    with pytest.raises(BackendError, match="device memory"):
        _nibble(ops, x, codes, scales, None, out, 64, 32)


_FIRST_CALLS = """
import sys, torch
from sys1rust_b200 import operators as ops
g = torch.Generator(device="cuda").manual_seed(1)
dev = dict(device="cuda")
x = torch.randn(3, 256, generator=g, **dev).half()
codes = torch.randint(0, 256, (64, 128), generator=g, dtype=torch.uint8, **dev)
scales = torch.rand(64, 2, generator=g, **dev).half()
y = torch.zeros(3, 64, dtype=torch.half, **dev)
page, heads, dim, count = 16, 2, 64, 300
kc, vc = torch.zeros(count, heads, page, dim, dtype=torch.int8, **dev), torch.zeros(count, heads, page, dim, dtype=torch.int8, **dev)
ks, vs = torch.zeros(count, heads, **dev), torch.zeros(count, heads, **dev)
cache = ops.Cache(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), count, page, heads, dim)
L = 4000
k, v = (torch.randn(L, heads * dim, generator=g, **dev).half() for _ in range(2))
rk, rv = torch.zeros_like(k), torch.zeros_like(v)
cu, zero, last = (torch.tensor(t, dtype=torch.int32, **dev) for t in ([0, L], [0], [L]))
table = torch.randperm(count, generator=g, **dev)[:250].int()
qs = {n: (torch.randn(n, 8 * dim, generator=g, **dev).half(), torch.zeros(n, 8 * dim, dtype=torch.half, **dev),
          torch.tensor([0, n], dtype=torch.int32, **dev)) for n in (1, 40)}
space = torch.zeros(max(ops.cache_attention_workspace(cache, 8, 1, n, L) for n in qs) + 16, dtype=torch.uint8, **dev)
logits = torch.randn(2, 5000, generator=g, **dev)
u = torch.rand(2, generator=g, **dev)
token = torch.zeros(2, dtype=torch.int32, **dev)

def run():
    st = torch.cuda.current_stream().cuda_stream
    ops.nibble_gemm(ops.DT_F16, x.data_ptr(), 256, codes.data_ptr(), 128, scales.data_ptr(), 2, y.data_ptr(), 64, 3, 64, 256, 128, stream=st)
    rows = (heads * dim, v.data_ptr(), heads * dim, cu.data_ptr(), zero.data_ptr(), table.data_ptr(), 250, 1, L)
    ops.cache_write(cache, ops.DT_F16, k.data_ptr(), *rows, stream=st)
    ops.cache_read(cache, ops.DT_F16, rk.data_ptr(), heads * dim, rv.data_ptr(), *rows[2:], stream=st)
    for n, (q, o, at) in qs.items():
        ops.cache_attention(cache, ops.DT_F16, q.data_ptr(), 8 * dim, o.data_ptr(), 8 * dim, 8, at.data_ptr(), last.data_ptr(),
                            table.data_ptr(), 250, 1, n, L, 0.125, workspace_ptr=space.data_ptr(), workspace_bytes=space.numel(), stream=st)
    ops.sample(ops.DT_F32, logits.data_ptr(), 5000, 2, 5000, token.data_ptr(), u.data_ptr(), stream=st)

outs = [y, kc, vc, ks, vs, rk, rv, token] + [o for _, o, _ in qs.values()]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()
graph.replay()
torch.cuda.synchronize()
captured = [t.clone() for t in outs]
for t in outs:
    t.zero_()
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, outs))
assert all(t.any() for t in outs)
"""


def test_first_calls_of_a_process_can_be_captured(ops):
    """Each operator's first call, which sets its kernels up, inside a stream capture; the replayed graph
    computes what the calls do."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]


@pytest.mark.parametrize("eager", [True, False])
def test_calls_behind_copies_fills_and_other_streams(ops, eager):
    """Inputs that a copy, a fill, a kernel of another stream and an operator made, one right before each
    call: a kernel that is scheduled early must still see all of them. Eagerly and as a replayed graph."""
    g = _gen(3)
    M, K = 4, 512
    _, codes, scales, _ = _nibble_inputs(M, K, K, 128, torch.float16, False, 4)
    src = [torch.randn(M, K, generator=g, device="cuda").half() * 0.1 for _ in range(20)]
    a, b, c = (torch.zeros(M, K, dtype=torch.float16, device="cuda") for _ in range(3))
    logits = torch.zeros(M, K, device="cuda")
    tokens = torch.zeros(20, M, dtype=torch.int32, device="cuda")
    sums = torch.zeros(20, M, K, device="cuda")
    u = torch.rand(M, generator=g, device="cuda")
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        for i in range(20):
            a.copy_(src[i])                                      # a copy, then the operator
            _nibble(ops, a, codes, scales, None, b, K, 128)
            _nibble(ops, b, codes, scales, None, c, K, 128)      # an operator behind an operator
            a.fill_(float("nan"))                                # overwritten right behind
            side.wait_stream(main)
            with torch.cuda.stream(side):
                logits.copy_(c)
                b.zero_()
            main.wait_stream(side)
            _nibble(ops, b, codes, scales, None, c, K, 128)      # behind another stream: zeros
            logits.add_(c)
            ops.sample(ops.DT_F32, logits.data_ptr(), K, M, K, tokens[i].data_ptr(), u.data_ptr(), stream=main.cuda_stream)
            sums[i].copy_(logits)
            logits.fill_(float("nan"))

    if eager:
        run()
    else:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graph.replay()
        tokens.zero_(), sums.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for i in range(20):
        b2, c2 = torch.empty_like(b), torch.empty_like(c)
        _nibble(ops, src[i], codes, scales, None, b2, K, 128)
        torch.cuda.synchronize()
        _nibble(ops, b2, codes, scales, None, c2, K, 128)
        torch.cuda.synchronize()
        want = c2.float()
        assert torch.equal(sums[i], want), i
        one = torch.zeros(M, dtype=torch.int32, device="cuda")
        ops.sample(ops.DT_F32, want.data_ptr(), K, M, K, one.data_ptr(), u.data_ptr(), stream=_stream())
        torch.cuda.synchronize()
        assert torch.equal(tokens[i], one), i


@pytest.mark.parametrize("eager", [True, False])
def test_gemm_whose_second_matrix_an_operator_wrote(ops, eager):
    """``s1c_gemm`` with few rows right behind the operator that writes its B: B is complete before it is
    loaded, eagerly and in a replayed graph. Bound: a rounded result and K products summed in fp32."""
    from sys1rust_b200 import backend
    M, N, K, inner, rounds = 16, 64, 2048, 8192, 20
    _, codes, scales, _ = _nibble_inputs(1, K, inner, 128, torch.bfloat16, False, 5)
    g = _gen(6)
    x = [(torch.randn(N, inner, generator=g, device="cuda") * 0.01).bfloat16() for _ in range(rounds)]
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    b = torch.zeros(N, K, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(rounds, M, N, dtype=torch.bfloat16, device="cuda")
    seen = torch.zeros(rounds, N, K, dtype=torch.bfloat16, device="cuda")

    def run():
        for i in range(rounds):
            _nibble(ops, x[i], codes, scales, None, b, inner, 128)
            backend.gemm(backend.EPI_STORE, a.data_ptr(), b.data_ptr(), out[i].data_ptr(), M, N, K, stream=_stream())
            seen[i].copy_(b)

    run()
    if not eager:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        out.zero_(), seen.zero_(), b.zero_()
        graph.replay()
    torch.cuda.synchronize()
    want = a.double() @ seen.double().transpose(1, 2)
    most = a.double().abs() @ seen.double().abs().transpose(1, 2)
    assert ((out.double() - want).abs() <= _u(torch.bfloat16) * want.abs() + (1 + 2.0 ** -8) * K * 2.0 ** -22 * most).all()


def test_gemm_with_few_rows_is_scheduled_while_the_kernel_before_it_ends(ops):
    """In a captured graph the edge into ``s1c_gemm``'s cluster kernel is a programmatic one, so that its set-up
    overlaps the end of the kernel before it."""
    import ctypes
    from sys1rust_b200 import backend
    M, N, K = 16, 64, 2048
    g = _gen(7)
    a, b = [torch.randn(r, K, generator=g, device="cuda").bfloat16() for r in (M, N)]
    out = torch.zeros(2, M, N, dtype=torch.bfloat16, device="cuda")

    def run():
        for o in out:
            backend.gemm(backend.EPI_STORE, a.data_ptr(), b.data_ptr(), o.data_ptr(), M, N, K, stream=_stream())

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        run()

    class Edge(ctypes.Structure):
        _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]

    get = ctypes.CDLL("libcudart.so.12").cudaGraphGetEdges_v2
    handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(8)
    ends, edges = [(ctypes.c_void_p * 8)() for _ in range(2)], (Edge * 8)()
    assert get(handle, ends[0], ends[1], edges, ctypes.byref(count)) == 0
    assert [e.type for e in edges[: count.value]] == [1]  # the one edge: programmatic
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and out.any()


@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_many_rows_and_gemms_share_the_tensor_memory(ops, D, eager):
    """Attention of many rows and ``s1c_gemm`` with few rows in turn, both in tensor memory and each scheduled while the
    one before it ends: B of the product is what the attention has written."""
    from sys1rust_b200 import backend
    H, G, rows, L, N, rounds = 2, 4, 64, 700, 16, 30
    c = Paged(ops, 1, L, H, D, 16, 95)
    K = H * G * D
    q = torch.randn(rows, K, generator=_gen(96), device="cuda").bfloat16()
    a = torch.randn(N, K, generator=_gen(97), device="cuda").bfloat16()
    att = torch.zeros(rounds, rows, K, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(rounds, N, rows, device="cuda")
    cu, ln = _i32([0, rows]), _i32([L])
    ws = torch.empty(max(1, ops.cache_attention_workspace(c.handle, H * G, 1, rows, L)), dtype=torch.uint8, device="cuda")

    def run():
        for i in range(rounds):
            ops.cache_attention(c.handle, ops.DT_BF16, q.data_ptr(), K, att[i].data_ptr(), K, H * G, cu.data_ptr(), ln.data_ptr(),
                                c.table.data_ptr(), c.table.shape[1], 1, rows, L, 0.1, workspace_ptr=ws.data_ptr(),
                                workspace_bytes=ws.numel(), stream=_stream())
            backend.gemm(backend.EPI_STORE, a.data_ptr(), att[i].data_ptr(), out[i].data_ptr(), N, rows, K, out_f32=True, stream=_stream())

    run()
    if not eager:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        att.zero_(), out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(att[0], x) for x in att) and all(torch.equal(out[0], x) for x in out)
    want = a.double() @ att[0].double().t()
    # K products summed in fp32
    assert ((out[0].double() - want).abs() <= K * 2.0 ** -22 * (a.double().abs() @ att[0].double().abs().t())).all() and want.any()
