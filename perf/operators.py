"""Cases, inputs and plain forms of the single-token operators.

Four operators that a host runs beside the encoder when it generates an answer token by token:

* ``nibble``  -- ``out = act(x W^T + bias)`` for a few rows x, W held as 4-bit codes with a scale
  (and optionally a zero point) for each group of columns of a row
* ``cache``   -- keys and values quantised to 8 bits as they are appended to a paged cache, one scale
  for each page and head, and rows read back from it
* ``attend``  -- causal attention of new rows over that cache: single tokens and pieces of prompts
* ``sample``  -- one token for each row of logits under temperature, top-k, top-p and min-p, from a
  given uniform number

``own`` chooses between the plain form (elementary torch operations) and the library's kernels.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODE = {"f32": 0, "f16": 1, "bf16": 2}  # the library's element types


def listed():
    return [
        # one token through a square projection of the encoder's width: launch latency counts
        dict(name="nibble_1x1024x1024", op="nibble", dtype="bf16", M=1, N=1024, K=1024, group=128, zeros=False, bias=False,
             act=0, out_f32=False),
        # one token through a wide feed-forward matrix: the weights' bytes count
        dict(name="nibble_1x28672x8192", op="nibble", dtype="f16", M=1, N=28672, K=8192, group=128, zeros=False, bias=False,
             act=0, out_f32=False),
        # sixteen sequences' logits over the encoder's vocabulary, from its feed-forward width (whose last group is short)
        dict(name="nibble_16x50368x2624", op="nibble", dtype="bf16", M=16, N=50368, K=2624, group=64, zeros=True, bias=True,
             act=0, out_f32=True),
        # a decode step: one new token in each of 64 sequences, the pages they land in read back
        dict(name="cache_decode_64", op="cache", dtype="bf16", n=64, new=1, start=4000, kv_heads=8, head_dim=128, page=16,
             rows=64, spread=1),
        # ragged prompts, the longest at the encoder's maximal length, behind odd starts; every row read back
        dict(name="cache_prompt_8192", op="cache", dtype="f16", n=8, new=8192, start=100, kv_heads=8, head_dim=128, page=64,
             rows=8192, spread=2),
        # a short run of tokens for a few sequences of the encoder's heads
        dict(name="cache_run_5", op="cache", dtype="bf16", n=3, new=5, start=37, kv_heads=16, head_dim=64, page=32, rows=40,
             spread=3),
        # one token of one short sequence, the encoder's heads
        dict(name="attend_1x700", op="attend", dtype="bf16", n=1, new=1, keys=700, heads=16, kv_heads=16, head_dim=64,
             page=16, window=-1, empty=False, spread=4),
        # a decode step of 64 ragged sequences with grouped heads, one of them not begun
        dict(name="attend_64x8192", op="attend", dtype="bf16", n=64, new=1, keys=8192, heads=32, kv_heads=8, head_dim=128,
             page=16, window=-1, empty=True, spread=5),
        # one token over a long document
        dict(name="attend_1x131072", op="attend", dtype="f16", n=1, new=1, keys=131072, heads=32, kv_heads=4, head_dim=128,
             page=64, window=-1, empty=False, spread=6),
        # pieces of prompts over what is cached of them
        dict(name="attend_prompt_4x512", op="attend", dtype="bf16", n=4, new=512, keys=4096, heads=16, kv_heads=4, head_dim=128,
             page=32, window=-1, empty=False, spread=7),
        # one sequence's next token over the encoder's vocabulary
        dict(name="sample_1x50368", op="sample", dtype="f32", rows=1, vocab=50368, temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0, masked=False),
        # a full batch's next tokens, nucleus and min-p, part of the vocabulary masked
        dict(name="sample_256x50368", op="sample", dtype="bf16", rows=256, vocab=50368, temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.02, masked=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["nibble", "cache", "attend", "sample"])
    half = rng.choice(["bf16", "f16"])
    if op == "nibble":
        M, K = _log(rng, 1, 64), _log(rng, 64, 8192)
        N = _log(rng, 64, max(64, min(60000, int(1.3e8 * 16 / max(M, 16) / K))))
        return dict(op=op, dtype=half, M=M, N=N, K=K, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.5, act=rng.choice([0, 1, 2]), out_f32=rng.random() < 0.3)
    if op == "cache":
        n, heads, dim = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128])
        new = _log(rng, 1, max(1, min(4096, int(2e7 / (n * heads * dim)))))
        start = _log(rng, 1, 5000) - 1
        return dict(op=op, dtype=half, n=n, new=new, start=start, kv_heads=heads, head_dim=dim, page=rng.choice([16, 32, 64]),
                    rows=rng.randint(1, min(new + start, new + 64)), spread=rng.randrange(1 << 20))
    if op == "attend":
        n, kv, dim = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        new = rng.choice([1, 1, _log(rng, 1, 16), _log(rng, 1, 512)])
        keys = _log(rng, 1, max(1, min(60000, int(2e8 / (n * kv * dim)), int(1e9 / (n * new * heads)))))
        return dict(op=op, dtype=half, n=n, new=new, keys=max(keys, new), heads=heads, kv_heads=kv, head_dim=dim,
                    page=rng.choice([16, 32, 64]), window=rng.choice([-1, -1, rng.randint(0, 3000)]),
                    empty=rng.random() < 0.3, spread=rng.randrange(1 << 20))
    rows = _log(rng, 1, 256)
    return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), rows=rows,
                vocab=_log(rng, 2, min(131072, int(1.2e7 / rows))), temperature=rng.choice([0.0, rng.uniform(0.3, 1.5)]),
                top_k=rng.choice([0, _log(rng, 1, 2000)]), top_p=rng.choice([1.0, rng.uniform(0.05, 0.99)]),
                min_p=rng.choice([0.0, rng.uniform(0.001, 0.3)]), masked=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------
# sizes that follow from a case alone


def _ragged(case, top, low):
    """n lengths in [low, top], the longest first; they belong to the case, not to the inputs."""
    r = random.Random(case["spread"])
    return [top] + [r.randint(low, top) for _ in range(case["n"] - 1)]


def _cache_sizes(case):
    """(new tokens, starts, rows read) of each sequence. The rows read are the last ones."""
    new = _ragged(case, case["new"], 1 if case["new"] == 1 else (case["new"] + 1) // 2)
    start = [max(0, case["start"] - 3 * i) for i in range(case["n"])]
    rows = [min(case["rows"], s + c) for s, c in zip(start, new)]
    return new, start, rows


def _attend_sizes(case):
    """(queries, keys) of each sequence; the queries are the last rows of the keys."""
    keys = _ragged(case, case["keys"], (case["keys"] + 1) // 2)
    new = [min(case["new"], k) for k in keys]
    if case["empty"] and case["n"] > 1:
        keys[-1] = 0  # a sequence that holds nothing yet: its row's mask leaves no key
    return new, keys


def work(case):
    if case["op"] == "nibble":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"])
        b = N * K / 2 + N * groups * 2 * (2 if case["zeros"] else 1) + M * K * 2 + M * N * (4 if case["out_f32"] else 2)
        return {"bytes": b + (4 * N if case["bias"] else 0), "flops": 2.0 * M * N * K}
    if case["op"] == "cache":
        new, start, rows = _cache_sizes(case)
        row = case["kv_heads"] * case["head_dim"] * 2  # values of K and V in one row
        # new rows read and their codes written; codes read and values written; a scale for each page touched
        pages = sum(-(-(s + c) // case["page"]) - s // case["page"] for s, c in zip(start, new))
        return {"bytes": sum(new) * row * 3 + sum(rows) * row * 3 + pages * case["kv_heads"] * 2 * 4, "flops": 3.0 * row * (sum(new) + sum(rows))}
    if case["op"] == "attend":
        new, keys = _attend_sizes(case)
        w, read, pairs = case["window"], 0, 0
        for c, k in zip(new, keys):
            if k:
                read += k if w < 0 else min(k, c + w)
                pairs += sum(p + 1 if w < 0 else min(p, w) + 1 for p in range(k - c, k))
        row = case["kv_heads"] * case["head_dim"] * 2
        b = read * row + read / case["page"] * case["kv_heads"] * 2 * 4 + sum(new) * case["heads"] * (case["head_dim"] * 4 + 4)
        return {"bytes": b, "flops": 4.0 * case["head_dim"] * case["heads"] * pairs}
    return {"bytes": case["rows"] * (case["vocab"] * (4 if case["dtype"] == "f32" else 2) + 28.0), "flops": 4.0 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------
# inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    cu = [0]
    cu.extend(sum(lens[: i + 1]) for i in range(len(lens)))
    return _ints(cu)


def _pages(case, g, longest):
    """A page table [n, ceil(longest / page)] over shuffled pages, with some pages that nobody uses."""
    per = max(1, -(-longest // case["page"]))
    count = case["n"] * per + 3
    table = torch.randperm(count, generator=g, device="cuda")[: case["n"] * per].view(case["n"], per).to(torch.int32)
    return table.contiguous(), count


def prepare(case, seed):
    g = _generator(seed)
    dt = _DT[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "nibble":
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        pitch = -(-K // 32) * 16  # bytes of a row of codes
        groups = -(-K // group)
        s["x"] = torch.randn(M, K, generator=g, device="cuda").to(dt)
        s["codes"] = torch.randint(0, 256, (N, pitch), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(N, groups, generator=g, device="cuda")) * (0.2 / math.sqrt(K))).to(dt)
        s["zeros"] = torch.randint(0, 16, (N, groups), generator=g, device="cuda").to(dt) if case["zeros"] else None
        s["bias"] = torch.randn(N, generator=g, device="cuda") if case["bias"] else None
        s["out"] = torch.empty(M, N, dtype=torch.float32 if case["out_f32"] else dt, device="cuda")
        return s
    if case["op"] == "cache":
        new, start, rows = _cache_sizes(case)
        H, D = case["kv_heads"], case["head_dim"]
        s["table"], count = _pages(case, g, max(a + b for a, b in zip(start, new)))
        shape = (count, H, case["page"], D)
        for name in ("k", "v"):
            s[name] = torch.randn(sum(new), H, D, generator=g, device="cuda").to(dt)
            s[name + "_codes"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            s[name + "_scales"] = (0.3 + torch.rand(count, H, generator=g, device="cuda")) * (3.0 / 127)
            s[name + "_rows"] = torch.empty(sum(rows), H, D, dtype=dt, device="cuda")
        s["cu"], s["start"] = _offsets(new), _ints(start)
        s["cu_rows"], s["first"] = _offsets(rows), _ints([a + c - r for a, c, r in zip(start, new, rows)])
        s["max_new"], s["max_rows"] = max(new), max(rows)
        s["cache"] = _handle(s, case, count)
        return s
    if case["op"] == "attend":
        new, keys = _attend_sizes(case)
        H, D = case["kv_heads"], case["head_dim"]
        s["table"], count = _pages(case, g, case["keys"])
        for name in ("k", "v"):
            # codes of normally distributed rows whose largest value stands at the end of the range
            normal = torch.randn(count, H, case["page"], D, generator=g, device="cuda", dtype=dt) * 32
            s[name + "_codes"] = normal.round().clamp(-127, 127).to(torch.int8)
            s[name + "_scales"] = (0.6 + 0.8 * torch.rand(count, H, generator=g, device="cuda")) / 32
            del normal
        s["q"] = torch.randn(sum(new), case["heads"], D, generator=g, device="cuda").to(dt)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(sum(new), case["heads"], device="cuda")
        s["cu"], s["len"] = _offsets(new), _ints(keys)
        s["max_q"], s["max_kv"] = max(new), max(keys)
        s["cache"] = _handle(s, case, count)
        s["workspace"] = _workspace(s, case)
        return s
    R, V = case["rows"], case["vocab"]
    x = torch.randn(R, V, generator=g, device="cuda") * 2.5
    if case["masked"]:
        x.masked_fill_(torch.rand(R, V, generator=g, device="cuda") < 0.1, float("-inf"))
    s["logits"] = x.to(dt)
    s["uniform"] = torch.rand(R, generator=g, device="cuda")
    s["temperature"] = torch.full((R,), case["temperature"], device="cuda")
    s["top_k"] = torch.full((R,), case["top_k"], dtype=torch.int32, device="cuda")
    s["top_p"] = torch.full((R,), case["top_p"], device="cuda")
    s["min_p"] = torch.full((R,), case["min_p"], device="cuda")
    s["token"] = torch.empty(R, dtype=torch.int32, device="cuda")
    s["prob"] = torch.empty(R, device="cuda")
    return s


def _handle(s, case, count):
    """The library's description of a cache, which a program keeps; the plain form needs none."""
    if own:
        from sys1rust_b200.operators import Cache
        return Cache(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(), s["v_scales"].data_ptr(),
                     count, case["page"], case["kv_heads"], case["head_dim"])
    return None


def _workspace(s, case):
    if own:
        from sys1rust_b200.operators import cache_attention_workspace
        return torch.empty(cache_attention_workspace(s["cache"], case["heads"], case["n"], s["max_q"], s["max_kv"]),
                           dtype=torch.uint8, device="cuda")
    return None


# ---------------------------------------------------------------------------------------------
# one pass


def run(state):
    if own:
        return _run_own(state)
    return {"nibble": _nibble, "cache": _cache, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


def _run_own(s):
    from sys1rust_b200 import operators as ops
    c = s["case"]
    dt, stream = _CODE[c["dtype"]], torch.cuda.current_stream().cuda_stream
    if c["op"] == "nibble":
        x, out, zeros, bias = s["x"], s["out"], s["zeros"], s["bias"]
        ops.nibble_gemm(dt, x.data_ptr(), x.stride(0), s["codes"].data_ptr(), s["codes"].stride(0), s["scales"].data_ptr(),
                        s["scales"].stride(0), out.data_ptr(), out.stride(0), c["M"], c["N"], c["K"], c["group"],
                        zeros_ptr=0 if zeros is None else zeros.data_ptr(), bias_ptr=0 if bias is None else bias.data_ptr(),
                        act=c["act"], out_f32=c["out_f32"], stream=stream)
        return out
    if c["op"] == "cache":
        k, v, kr, vr, table = s["k"], s["v"], s["k_rows"], s["v_rows"], s["table"]
        ops.cache_write(s["cache"], dt, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), s["cu"].data_ptr(),
                        s["start"].data_ptr(), table.data_ptr(), table.shape[1], c["n"], s["max_new"], stream=stream)
        ops.cache_read(s["cache"], dt, kr.data_ptr(), kr.stride(0), vr.data_ptr(), vr.stride(0), s["cu_rows"].data_ptr(),
                       s["first"].data_ptr(), table.data_ptr(), table.shape[1], c["n"], s["max_rows"], stream=stream)
        return {"k": kr, "v": vr, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if c["op"] == "attend":
        q, out, table = s["q"], s["out"], s["table"]
        ops.cache_attention(s["cache"], dt, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), c["heads"],
                            s["cu"].data_ptr(), s["len"].data_ptr(), table.data_ptr(), table.shape[1], c["n"], s["max_q"],
                            s["max_kv"], 1 / math.sqrt(c["head_dim"]), window=c["window"], lse_ptr=s["lse"].data_ptr(),
                            workspace_ptr=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=stream)
        return {"out": out, "lse": s["lse"]}
    ops.sample(dt, s["logits"].data_ptr(), s["logits"].stride(0), c["rows"], c["vocab"], s["token"].data_ptr(),
               s["uniform"].data_ptr(), temperature_ptr=s["temperature"].data_ptr(), top_k_ptr=s["top_k"].data_ptr(),
               top_p_ptr=s["top_p"].data_ptr(), min_p_ptr=s["min_p"].data_ptr(), prob_ptr=s["prob"].data_ptr(), stream=stream)
    return {"token": s["token"], "prob": s["prob"]}


# ---------------------------------------------------------------------------------------------
# plain forms


def _weights(s, dtype):
    """The matrix [N, K] that codes, scales and zero points stand for: scale * (code - zero), zero 8 where none is given."""
    K, group = s["case"]["K"], s["case"]["group"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(1)[:, :K].to(dtype)
    at = torch.arange(K, device="cuda") // group
    zero = s["zeros"].to(dtype)[:, at] if s["zeros"] is not None else 8.0
    return (codes - zero) * s["scales"].to(dtype)[:, at]


def _nibble(s):
    y = s["x"].float() @ _weights(s, torch.float32).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    if act == 1:
        y = torch.clamp(y, min=0)
    if act == 2:
        y = y * 0.5 * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(s["out"].dtype)


def _cache(s):
    c = s["case"]
    n, P = c["n"], c["page"]
    cu, start, table = s["cu"].long(), s["start"].long(), s["table"].long()
    count = cu[1:] - cu[:-1]
    units = (s["max_new"] + P - 2) // P + 1  # pages that one sequence's new rows can touch
    page = start[:, None] // P + torch.arange(units, device="cuda")  # [n, units], by its place in the table
    used = page * P < (start + count)[:, None]
    where = table.gather(1, page.clamp(max=table.shape[1] - 1))[used]  # pages written
    at = (page[:, :, None] * P + torch.arange(P, device="cuda"))[used]  # positions of their rows, [pages, P]
    seq = torch.arange(n, device="cuda")[:, None].expand(n, units)[used]
    old = (at < start[seq][:, None])[:, None, :, None]
    fresh = ((at >= start[seq][:, None]) & (at < (start + count)[seq][:, None]))[:, None, :, None]
    row = (cu[seq] - start[seq])[:, None] + at
    out = {}
    for name in ("k", "v"):
        x, codes, scales = s[name], s[name + "_codes"], s[name + "_scales"]
        new = x[row.clamp(0, x.shape[0] - 1)].double().transpose(1, 2) * fresh  # [pages, H, P, D]
        had = torch.where(old.any(2)[:, :, 0], scales[where], 0.0)
        scale = torch.maximum(had, (new.abs().amax((2, 3)) / 127).float())
        div = torch.where(scale > 0, scale, 1.0).double()[:, :, None, None]
        was = codes[where]
        again = (was.double() * had.double()[:, :, None, None] / div).round()
        codes[where] = torch.where(fresh, (new / div).round(), torch.where(old, again, was.double())).to(torch.int8)
        scales[where] = scale
        out[name + "_scales"] = scales
        out[name] = _rows(s, name).to(x.dtype)
    return out


def _rows(s, name):
    """The rows that the case reads back."""
    cu, first, table, P = s["cu_rows"].long(), s["first"].long(), s["table"].long(), s["case"]["page"]
    i = torch.arange(s[name + "_rows"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, i, right=True) - 1
    at = first[seq] + i - cu[seq]
    page = table[seq, at // P]
    return s[name + "_codes"][page, :, at % P].float() * s[name + "_scales"][page][:, :, None]


def _attend(s):
    c = s["case"]
    n, H, G, D, Q = c["n"], c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"], s["max_q"]
    cu, length = s["cu"].long(), s["len"].long()
    count = cu[1:] - cu[:-1]
    i = torch.arange(Q, device="cuda")
    q = s["q"][(cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)].float().view(n, Q, H, G, D)
    k, v = [(s[x + "_codes"][s["table"].long()].float() * s[x + "_scales"][s["table"].long()][..., None, None])
            .transpose(2, 3).reshape(n, -1, H, D) for x in ("k", "v")]  # [n, keys, H, D]
    score = torch.einsum("nqhgd,nkhd->nhgqk", q, k) / math.sqrt(D)
    at = (length - count)[:, None] + i  # positions of the queries
    key = torch.arange(k.shape[1], device="cuda")
    seen = (key <= at[..., None]) & (key < length[:, None, None])
    if c["window"] >= 0:
        seen = seen & (key >= at[..., None] - c["window"])
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("nhgqk,nkhd->nqhgd", p, v) / total.permute(0, 3, 1, 2, 4).clamp(min=1e-30)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2)
    real = i < count[:, None]
    return {"out": o.reshape(n, Q, H * G, D)[real].to(s["q"].dtype), "lse": lse.reshape(n, Q, H * G)[real]}


def _sample(s):
    x = s["logits"].double()
    R, V = x.shape
    top = x.amax(1, keepdim=True)
    T = s["temperature"].double()[:, None]
    z = torch.where(T > 0, (x - top) / torch.where(T > 0, T, 1.0), torch.where(x == top, 0.0, -math.inf))
    e = torch.exp(z)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    es = e.gather(1, order)
    rank = torch.arange(V, device="cuda")
    k = torch.where(T[:, 0] > 0, torch.where(s["top_k"] > 0, s["top_k"], V), 1)[:, None]
    es = es * (rank < k)
    before = torch.cumsum(es, 1)
    goal = s["top_p"].double()[:, None] * before[:, -1:]
    before = torch.nn.functional.pad(before[:, :-1], (1, 0))
    keep = (rank == 0) | ((before < goal) | (s["top_p"][:, None] >= 1)) & (es >= s["min_p"].double()[:, None].clamp(max=1.0))
    mass = torch.zeros_like(e).scatter_(1, order, es * keep)
    along = torch.cumsum(mass, 1)
    total = along[:, -1:]
    token = (along <= s["uniform"].double()[:, None] * total).sum(1, keepdim=True)
    last = (mass > 0).long().mul(rank + 1).amax(1, keepdim=True) - 1
    token = torch.minimum(token, last)
    return {"token": token[:, 0].to(torch.int32), "prob": (mass.gather(1, token) / total)[:, 0].float()}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"nibble": _exact_nibble, "cache": _exact_cache, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)


def _exact_nibble(case, s):
    M, N, K, group = case["M"], case["N"], case["K"], case["group"]
    x = s["x"].double()
    y = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for g in range(-(-K // group)):  # group by group: scale * (sum x code - zero * sum x)
        lo, hi = g * group, min(K, (g + 1) * group)
        packed = s["codes"][:, lo // 2: (hi + 1) // 2].int()
        code = torch.empty(N, packed.shape[1] * 2, dtype=torch.float64, device="cuda")
        code[:, 0::2], code[:, 1::2] = packed % 16, packed // 16
        zero = 8.0 if s["zeros"] is None else s["zeros"][:, g].double()
        y += s["scales"][:, g].double() * (x[:, lo:hi] @ code[:, : hi - lo].t() - zero * x[:, lo:hi].sum(1, keepdim=True))
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == 1:
        y = torch.relu(y)
    if case["act"] == 2:
        y = torch.special.ndtr(y) * y
    return y


def _exact_cache(case, s):
    new, start, rows = _cache_sizes(case)
    P, table = case["page"], s["table"].cpu()
    out = {}
    for name in ("k", "v"):
        codes, scales, x = s[name + "_codes"].double(), s[name + "_scales"].double(), s[name].double()
        base, took = 0, []
        for i, (c, a, r) in enumerate(zip(new, start, rows)):
            for p in range(a // P, -(-(a + c) // P)):
                lo, hi, page = max(a, p * P), min(a + c, (p + 1) * P), int(table[i, p])
                part = x[base + lo - a: base + hi - a].transpose(0, 1)  # [H, rows, D]
                keep = lo - p * P
                # the definition holds the scale in 32 bits
                scale = (part.abs().amax((1, 2)) / 127).float().double()
                if keep:
                    scale = torch.maximum(scale, scales[page])
                    codes[page, :, :keep] = (codes[page, :, :keep] * (scales[page] / scale)[:, None, None]).round()
                codes[page, :, keep: keep + hi - lo] = (part / scale[:, None, None]).round()
                scales[page] = scale
            base += c
            at = torch.arange(a + c - r, a + c)
            pages = table[i][at // P].long().cuda()
            took.append(codes[pages, :, (at % P).cuda()] * scales[pages][:, :, None])
        out[name], out[name + "_scales"] = torch.cat(took), scales
    return out


def _exact_attend(case, s):
    new, keys = _attend_sizes(case)
    H, G, D, P, w = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"], case["page"], case["window"]
    out, lse, base = [], [], 0
    for i, (c, L) in enumerate(zip(new, keys)):
        q = s["q"][base: base + c].double().view(c, H, G, D)
        base += c
        pages = s["table"][i, : -(-L // P)].long()
        kv = [(s[x + "_codes"][pages].double() * s[x + "_scales"][pages].double()[..., None, None]).transpose(0, 1).reshape(H, len(pages) * P, D)[:, :L]
              for x in ("k", "v")]
        at = torch.arange(L - c, L, device="cuda")[:, None]
        key = torch.arange(L, device="cuda")[None]
        hide = (key > at) | ((key < at - w) if w >= 0 else False)
        for h in range(H):
            a = (q[:, h].reshape(c * G, D) @ kv[0][h].t() / math.sqrt(D)).view(c, G, L).masked_fill(hide[:, None], -math.inf)
            lse.append(torch.logsumexp(a, -1))  # [c, G]; of no key: -inf
            out.append(torch.softmax(a, -1).nan_to_num(0.0).view(c * G, L) @ kv[1][h])
        out[-H:] = [torch.stack([o.view(c, G, D) for o in out[-H:]], 1).reshape(c, H * G, D)]
        lse[-H:] = [torch.stack(lse[-H:], 1).reshape(c, H * G)]
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _exact_sample(case, s):
    import numpy as np
    tokens, probs = [], []
    for r in range(case["rows"]):
        x, u = s["logits"][r].double().cpu().numpy(), float(s["uniform"][r])
        T, k, p, m = (float(s[name][r]) for name in ("temperature", "top_k", "top_p", "min_p"))
        if T <= 0:
            tokens.append(int(x.argmax()))
            probs.append(1.0)
            continue
        e = np.exp((x - x.max()) / T)
        order = np.lexsort((np.arange(x.size), -x))
        if k > 0:
            order = order[: int(k)]
        if p < 1:
            cum = np.cumsum(e[order])
            order = order[: int(np.searchsorted(cum, p * cum[-1], side="left")) + 1]
        order = order[e[order] >= min(m, 1.0)]
        order.sort()
        cum = np.cumsum(e[order])
        j = min(int(np.searchsorted(cum, u * cum[-1], side="right")), order.size - 1)
        tokens.append(int(order[j]))
        probs.append(float(e[order[j]] / cum[-1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}
