"""The 8-bit paged KV cache on the GPU: the store and the three attentions against 64-bit formulas.

Tolerances.  Attention: the codes are exact as halves, scores are fp32 sums of 128 products, the
probabilities are rounded to halves (2^-11 each) and the output to bf16 (2^-8), so an output element
is off by at most 2^-8 |o| + e * sum_j p_j |v_j|, with e = 2^-11 for the probabilities and as much again
for the scores: their error is at most 128 * 2^-24 * scale * sum_d |q_d k_d|, under 2^-11 for sums up to
64 (the cases' are below 40; `attention_tol` adds the term where a case goes beyond).
Store: fp32 arithmetic before one rounding to e4m3, so a code is within half a step of the 64-bit
quotient plus 2^-18 of the head row's largest value.
"""
import math

import numpy as np
import pytest
import torch

from qwen3_naive_inference_b200 import ops

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
D, PAGE, BLOCK = 128, 256, 64


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------ helpers
def random_cache(g, num_blocks, hkv):
    """CPU caches: random finite codes, scales of several powers of two."""
    out = []
    for _ in range(2):
        x = torch.randn(num_blocks, hkv, PAGE, D, generator=g) * 100
        out.append(x.clamp(-448, 448).to(F8))
    for _ in range(2):
        out.append(torch.exp2(torch.randint(-7, -4, (num_blocks, hkv, 4), generator=g).float()))
    return out


def values(codes, scales):
    return (codes.double().view(*scales.shape, BLOCK, D) * scales.double()[..., None, None]).view(codes.shape)


def rows_of(cache64, pages, a, b, h):
    """Keys [a, b) of one head, [b - a, D] in 64 bits, from a list of page ids."""
    j = torch.arange(a, b)
    return cache64[torch.as_tensor(pages)[j // PAGE].long(), h, j % PAGE]


def attend(q, parts, scale, past=None):
    """One sequence, one q head: q [n, D] over the keys and values of `parts` [(k, v)]; with `past` row i
    sees the first past + i + 1 keys.  Returns (o, sum_j p_j |v_j|, largest sum_d |q_d k_d|)."""
    k, v = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    if k.shape[0] == 0:
        z = torch.zeros(q.shape[0], D, dtype=torch.float64)
        return z, z, 0.0
    x = q.double() @ k.T * scale
    if past is not None:
        x = x.masked_fill(torch.arange(k.shape[0]) > past + torch.arange(q.shape[0])[:, None], -math.inf)
    p = torch.softmax(x, -1)
    return p @ v, p @ v.abs(), float((q.double().abs() @ k.abs().T).max() * scale)


def check_attention(out, ref, mag, most, msg=""):
    e = 2.0 ** -11 + 128 * 2.0 ** -24 * max(64.0, most)
    tol = 2.0 ** -8 * ref.abs() + e * mag + 1e-30
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all(), msg
    bad = (err > tol).nonzero()
    assert not len(bad), f"{msg} {len(bad)} beyond, first {bad[0].tolist()}: {err[tuple(bad[0])]} > {tol[tuple(bad[0])]}"


def paged(g, lens, num_blocks, width=None, fill=-1):
    """Random page tables for sequences of `lens` tokens."""
    pages = [-(-n // PAGE) for n in lens]
    assert sum(pages) <= num_blocks
    pool = torch.randperm(num_blocks, generator=g).tolist()
    table = torch.full((len(lens), width or max(1, max(pages))), fill, dtype=torch.int32)
    for i, n in enumerate(pages):
        for w in range(n):
            table[i, w] = pool.pop()
    return table


def spoil_dead(k, v, table, lens):
    """NaN codes in every row behind the end of a sequence's last page: they may not reach an output."""
    for i, n in enumerate(lens):
        if n % PAGE:
            page = int(table[i, n // PAGE])
            for c in (k, v):
                c.view(torch.uint8)[page, :, n % PAGE:] = 0x7F


def on(dev, *ts):
    return [t.to(dev) for t in ts]


# ------------------------------------------------------------------------------------------ decode
DECODE = [
    # hq, hkv, context lengths (keys = context + 1; -1: none)
    (16, 8, [0]), (16, 8, [62, 63, 64, 65]), (16, 8, [254, 255, 256, 257, 300]),
    (16, 8, [-1, 700, -1, 1]), (4, 2, [1000, 3, 4095]), (8, 8, [513, 77]), (32, 8, [130, 2047]),
    (40, 8, [90, 600]), (16, 1, [300, 0, 64]), (32, 2, [777]), (2, 1, [9000]), (14, 2, [128, 127, 640]),
]


@pytest.mark.parametrize("hq,hkv,ctx", DECODE)
@pytest.mark.parametrize("split", [None, 64, 320])
def test_decode(cuda, hq, hkv, ctx, split):
    g = gen(len(ctx) * 100 + hq)
    lens = [c + 1 for c in ctx]
    nb = sum(-(-n // PAGE) for n in lens) + 2
    k, v, ks, vs = random_cache(g, nb, hkv)
    table = paged(g, lens, nb)
    spoil_dead(k, v, table, lens)
    q = torch.randn(len(lens), hq, D, generator=g).to(BF)
    scale = D ** -0.5
    args = on(cuda, q, k, v, ks, vs, table, torch.tensor(ctx, dtype=torch.int32))
    if split is None:
        out = ops.paged_decode_attention_fp8(*args, scale)
    else:
        out = ops.paged_decode_attention_fp8(*args, scale, split_tokens=split, max_splits=-(-max(lens) // split))
    k64, v64 = values(k, ks), values(v, vs)
    for b, n in enumerate(lens):
        for h in range(hq):
            kv = [(rows_of(c, table[b], 0, n, h // (hq // hkv))) for c in (k64, v64)]
            ref, mag, most = attend(q[b, h:h + 1], [kv], scale)
            check_attention(out[b, h:h + 1], ref, mag, most, f"row {b} head {h}")
    ops.check_device_errors()


def test_decode_rows_apart_and_reused_output(cuda):
    """Query rows inside a wider tensor, a caller's output and workspace, max_ctx above the lengths."""
    g = gen(5)
    lens = [200, 1100, 64]
    k, v, ks, vs = random_cache(g, 12, 4)
    table = paged(g, lens, 12, width=9)
    wide = torch.randn(3, 24, D, generator=g).to(BF)
    q = wide[:, 4:12]
    args = on(cuda, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32))
    qd = wide.to(cuda)[:, 4:12]
    out = torch.full((3, 8, D), 7.0, dtype=BF, device=cuda)
    ws = ops.workspace_fp8(3, 8, 32, cuda).fill_(math.nan)
    got = ops.paged_decode_attention_fp8(qd, *args, 0.1, seqlen_add=0, split_tokens=128, max_splits=32, workspace=ws,
                                         out=out)
    assert got is out
    plain = ops.paged_decode_attention_fp8(qd.contiguous(), *args, 0.1, seqlen_add=0, max_ctx=2304)
    k64, v64 = values(k, ks), values(v, vs)
    for b, n in enumerate(lens):
        for h in range(8):
            ref, mag, most = attend(q[b, h:h + 1], [[rows_of(c, table[b], 0, n, h // 2) for c in (k64, v64)]], 0.1)
            check_attention(out[b, h:h + 1], ref, mag, most)
            check_attention(plain[b, h:h + 1], ref, mag, most)
    ops.check_device_errors()


def test_decode_bad_pages_are_reported(cuda):
    """A page outside the pool, a missing one and a table that is too narrow: reported, the keys left out."""
    g = gen(6)
    k, v, ks, vs = random_cache(g, 4, 2)
    q = torch.randn(1, 4, D, generator=g).to(BF)
    k64, v64 = values(k, ks), values(v, vs)
    for table in ([[1, 4, 2]], [[1, -1, 2]], [[1, 1 << 30, 2]]):
        t = torch.tensor(table, dtype=torch.int32)
        args = on(cuda, q, k, v, ks, vs, t, torch.tensor([599], dtype=torch.int32))
        out = ops.paged_decode_attention_fp8(*args, 0.1)
        with pytest.raises(ops.NativeError, match="page id"):
            ops.check_device_errors()
        for h in range(4):
            parts = [[rows_of(c, [1], 0, 256, h // 2) for c in (k64, v64)],
                     [rows_of(c, [2], 0, 88, h // 2) for c in (k64, v64)]]
            check_attention(out[0, h:h + 1], *attend(q[0, h:h + 1], parts, 0.1))
    args = on(cuda, q, k, v, ks, vs, torch.tensor([[1]], dtype=torch.int32), torch.tensor([299], dtype=torch.int32))
    ops.paged_decode_attention_fp8(*args, 0.1, max_ctx=512)
    with pytest.raises(ops.NativeError, match="page id"):
        ops.check_device_errors()
    ops.check_device_errors()


@pytest.mark.parametrize("keys,max_ctx", [(1000, 512), (3000, 2000)])
def test_decode_keys_beyond_max_ctx_are_reported(cuda, keys, max_ctx):
    """A sequence longer than max_ctx, in one split (which has no workspace) and in several: reported, the
    output that of the keys the plan covers; its neighbours are not touched by it."""
    g = gen(11)
    k, v, ks, vs = random_cache(g, 14, 2)
    table = paged(g, [keys, 70], 14)
    q = torch.randn(2, 4, D, generator=g).to(BF)
    split, n = ops.decode_split_plan_fp8(2, 2, max_ctx)
    assert (n == 1) == (max_ctx <= 768) and split * n < keys
    args = on(cuda, q, k, v, ks, vs, table, torch.tensor([keys, 70], dtype=torch.int32))
    out = ops.paged_decode_attention_fp8(*args, 0.1, seqlen_add=0, max_ctx=max_ctx)
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    k64, v64 = values(k, ks), values(v, vs)
    for b, seen in enumerate((split * n, 70)):
        for h in range(4):
            kv = [rows_of(c, table[b], 0, seen, h // 2) for c in (k64, v64)]
            check_attention(out[b, h:h + 1], *attend(q[b, h:h + 1], [kv], 0.1), f"row {b} head {h}")


def test_decode_scales_far_apart(cuda):
    """Blocks whose scales differ by 2^60, and whose values are zero under the smallest scale: each block's
    share counts whatever its neighbours hold."""
    g = gen(7)
    k, v, ks, vs = random_cache(g, 3, 1)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    q = torch.randn(1, 2, D, generator=g).to(BF)
    n = 700
    for case in range(3):
        vs2, v2 = vs.clone(), v.clone()
        if case == 0:
            vs2[2, 0, 1], vs2[0, 0, 2] = 2.0 ** 30, 2.0 ** -30
        elif case == 1:  # all but one block of V zero under the smallest scale
            vs2[:] = 2.0 ** -126
            v2.view(torch.uint8)[:] = 0
            vs2[0, 0, 1] = 2.0 ** -40
            v2[0, :, 64:128] = v[0, :, 64:128]
        else:
            vs2[:] = 2.0 ** -100
        args = on(cuda, q, k, v2, ks, vs2, table, torch.tensor([n - 1], dtype=torch.int32))
        out = ops.paged_decode_attention_fp8(*args, 0.02)
        pre = ops.attention_paged_prefill_fp8(args[0], *args[1:5], *on(cuda, torch.tensor([0, 1], dtype=torch.int32),
                                              torch.tensor([0, n], dtype=torch.int32)), 1, args[5], 0.02)
        k64, v64 = values(k, ks), values(v2, vs2)
        for h in range(2):
            ref = attend(q[0, h:h + 1], [[rows_of(c, table[0], 0, n, 0) for c in (k64, v64)]], 0.02)
            check_attention(out[0, h:h + 1], *ref, f"case {case}")
            check_attention(pre[0, h:h + 1], *ref, f"prefill, case {case}")


def test_decode_large_queries(cuda):
    """Queries far beyond the range of a half keep their bf16 precision."""
    g = gen(8)
    k, v, ks, vs = random_cache(g, 2, 2)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    for big in (1e20, 1e-20):
        q = (torch.randn(1, 8, D, generator=g) * big).to(BF)
        scale = 0.05 / big
        args = on(cuda, q, k, v, ks, vs, table, torch.tensor([399], dtype=torch.int32))
        out = ops.paged_decode_attention_fp8(*args, scale)
        pre = ops.attention_paged_prefill_fp8(args[0], *args[1:5], *on(cuda, torch.tensor([0, 1], dtype=torch.int32),
                                              torch.tensor([0, 400], dtype=torch.int32)), 1, args[5], scale)
        k64, v64 = values(k, ks), values(v, vs)
        for h in range(8):
            ref = attend(q[0, h:h + 1], [[rows_of(c, table[0], 0, 400, h // 4) for c in (k64, v64)]], scale)
            check_attention(out[0, h:h + 1], *ref)
            check_attention(pre[0, h:h + 1], *ref)


@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_scales_that_are_not_positive(cuda, scale):
    """A negative softmax scale turns the order of the scores, a scale of zero gives the mean of V."""
    g = gen(9)
    k, v, ks, vs = random_cache(g, 2, 2)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    q = torch.randn(140, 8, D, generator=g).to(BF)
    args = on(cuda, q, k, v, ks, vs, table)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    dec = ops.paged_decode_attention_fp8(args[0][:1], *args[1:], i32(449), scale)
    pre = ops.attention_paged_prefill_fp8(*args[:5], i32(0, 140), i32(0, 500), 140, args[5], scale)
    k64, v64 = values(k, ks), values(v, vs)
    for h in range(8):
        kv = [rows_of(c, table[0], 0, 500, h // 4) for c in (k64, v64)]
        check_attention(pre[:, h], *attend(q[:, h], [kv], scale, 360))
        check_attention(dec[:, h], *attend(q[:1, h], [[c[:450] for c in kv]], scale))


def test_values_that_are_not_finite_in_queries(cuda):
    """NaN and infinities in one row's queries stay in that row."""
    g = gen(10)
    k, v, ks, vs = random_cache(g, 2, 2)
    table = torch.tensor([[1, 0]] * 3, dtype=torch.int32)
    q = torch.randn(3, 4, D, generator=g).to(BF)
    bad = q.clone()
    bad[1, 2, 5], bad[1, 3, 0] = math.nan, math.inf
    args = on(cuda, k, v, ks, vs, table, torch.tensor([300, 299, 100], dtype=torch.int32))
    a, b = (ops.paged_decode_attention_fp8(x.to(cuda), *args, 0.1) for x in (q, bad))
    assert bool(b[1, 2].isnan().all()) and torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, :2], b[1, :2])
    cu = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    ck = torch.tensor([0, 400], dtype=torch.int32, device=cuda)
    a, b = (ops.attention_paged_prefill_fp8(x.to(cuda), *args[:4], cu, ck, 3, args[4][:1].contiguous(), 0.1) for x in (q, bad))
    assert bool(b[1, 2].isnan().all()) and torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, :2], b[1, :2])


# ------------------------------------------------------------------------------------------ grouped
GROUPED = [
    # hq, hkv, per group: shared keys, own keys of each member
    (16, 8, [(300, [1, 2, 70, 64, 65, 128, 300, 5]), (64, [9]), (1, [33, 1])]),
    (16, 8, [(0, [17, 300]), (255, [64] * 8)]),
    (4, 2, [(1500, [600, 3]), (256, [1, 1, 1])]),
    (32, 4, [(200, [10, 20, 30]), (70, [100] * 8)]),
    (40, 8, [(130, [7, 8, 9, 64])]),
    (16, 1, [(65, [3, 200])]),
    (8, 8, [(600, [1] * 8)]),
]


def grouped_inputs(g, hq, hkv, groups, dev):
    n = sum(len(o) for _, o in groups)
    nb = sum(-(-s // PAGE) + sum(-(-x // PAGE) for x in o) for s, o in groups) + 2
    pool = torch.randperm(nb, generator=g).tolist()
    k, v, ks, vs = random_cache(g, nb, hkv)
    width = max(-(-s // PAGE) + max(-(-x // PAGE) for x in o) for s, o in groups)
    table = torch.full((n, width), -1, dtype=torch.int32)
    members = torch.full((len(groups), 8), -1, dtype=torch.int32)
    lens, start, b, parts = [], [], 0, []
    order = torch.randperm(n, generator=g).tolist()  # group members are any rows
    for gi, (s, o) in enumerate(groups):
        head = [pool.pop() for _ in range(-(-s // PAGE))]
        donor = None
        for m, x in enumerate(o):
            row = order[b]
            pages = head + [pool.pop() for _ in range(-(-x // PAGE))]
            table[row, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            members[gi, m] = row
            donor = row if donor is None else donor
            st = len(head) * PAGE
            lens.append((row, st + x))
            start.append((row, st))
            parts.append((row, head, s, pages, st, st + x))
            for c in (k, v):  # what no row may see
                if x % PAGE:
                    c.view(torch.uint8)[pages[-1], :, x % PAGE:] = 0x7F
                if s % PAGE:
                    c.view(torch.uint8)[head[-1], :, s % PAGE:] = 0x7F
            b += 1
    flat = lambda pairs: torch.tensor([x for _, x in sorted(pairs)], dtype=torch.int32)  # noqa: E731
    q = torch.randn(n, hq, D, generator=g).to(BF)
    dev_args = on(dev, q, k, v, ks, vs, table, flat([(r, x - 1) for r, x in lens]))
    grp = on(dev, members, torch.tensor([s for s, _ in groups], dtype=torch.int32), flat(start))
    return q, k, v, ks, vs, parts, dev_args, grp


def test_grouped_table_with_empty_entries(cuda):
    """A table captured for any grouping: live groups anywhere in it, several to one CTA."""
    g = gen(50)
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, 16, 8, [(300, [5, 70, 64]), (600, [1, 2]), (64, [200] * 8), (90, [3])], cuda)
    n = q.shape[0]
    plan = ops.grouped_decode_plan_fp8(n, 4, 16, 8, 600, 200)
    want = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan)
    for step, at in ((41, [0, 1, 2, 3]), (4, [0, 1, 2, 3]), (6, [0, 6, 12, 18]), (5, [5, 17, 18, 40]), (1, [7, 0, 39, 20])):
        members = torch.full((41, 8), -1, dtype=torch.int32, device=cuda)
        shared = torch.zeros(41, dtype=torch.int32, device=cuda)
        for i, slot in enumerate(at):
            members[slot], shared[slot] = grp[0][i], grp[1][i]
        out = ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, shared, grp[2], (step, 64, 24, 128, 8))
        check = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, (2, 64, 24, 128, 8))
        assert torch.equal(out, check)
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -6, atol=1e-2)
    ops.check_device_errors()


@pytest.mark.parametrize("hq,hkv,groups", GROUPED)
@pytest.mark.parametrize("plan", [None, (2, 64, 24, 128, 8)])
def test_grouped(cuda, hq, hkv, groups, plan):
    g = gen(hq + len(groups))
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, hq, hkv, groups, cuda)
    if plan is None:
        plan = ops.grouped_decode_plan_fp8(q.shape[0], len(groups), hq, hkv, max(s for s, _ in groups),
                                           max(max(o) for _, o in groups))
    out = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan)
    k64, v64 = values(k, ks), values(v, vs)
    for row, head, s, pages, a, b in parts:
        for h in range(hq):
            kvh = h // (hq // hkv)
            p = [[rows_of(c, pages, a, b, kvh) for c in (k64, v64)]]
            if s:
                p.insert(0, [rows_of(c, head, 0, s, kvh) for c in (k64, v64)])
            check_attention(out[row, h:h + 1], *attend(q[row, h:h + 1], p, 0.1), f"row {row} head {h}")
    ops.check_device_errors()


def many_groups(g, n, top_shared, top_own):
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    return [(pick(1, top_shared), [pick(1, top_own) for _ in range(1 + i % 8)]) for i in range(n)]


@pytest.mark.parametrize("hq,hkv,n", [(16, 8, 50), (8, 8, 64), (40, 8, 8), (24, 8, 16), (96, 8, 8), (64, 8, 9)])
def test_grouped_many(cuda, hq, hkv, n):
    """Enough groups for a CTA to take members through all their keys: against the formula, and with a table
    that has more entries than there are groups, walked in steps."""
    g = gen(60 + hq)
    groups = many_groups(g, n, 150, 140)
    groups[0] = (130, [1, 64, 65, 63, 128, 2, 129, 140])
    groups[1] = (64, [64] * 8)
    groups[2] = (1, [1])
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, hq, hkv, groups, cuda)
    plan = ops.grouped_decode_plan_fp8(q.shape[0], n, hq, hkv, 150, 140)
    assert ops._grouped_whole(hq, hkv, n, *plan[1:]) and plan[1:] == (192, 1, 192, 1)
    out = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan, out=torch.full_like(args[0], 3.0))
    k64, v64 = values(k, ks), values(v, vs)
    for row, head, s, pages, st, end in parts:
        for h in (row % hq, hq - 1 - row % hq):
            kv = [[torch.cat([rows_of(c, head, 0, s, h // (hq // hkv)), rows_of(c, pages, st, end, h // (hq // hkv))])
                   for c in (k64, v64)]]
            check_attention(out[row, h:h + 1], *attend(q[row, h:h + 1], kv, 0.1), f"row {row} head {h}")
    big = 2 * n + 3
    members = torch.full((big, 8), -1, dtype=torch.int32, device=cuda)
    shared = torch.zeros(big, dtype=torch.int32, device=cuda)
    at = torch.randperm(big, generator=g)[:n].to(cuda)
    members[at], shared[at] = grp[0], grp[1]
    again = ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, shared, grp[2], plan)
    assert torch.equal(again, out)
    # the same keys split and joined
    split = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, (n, 64, 3, 64, 3))
    assert torch.allclose(split.float(), out.float(), rtol=2.0 ** -6, atol=1e-2)
    ops.check_device_errors()
    # a sequence in no group gets zeros, its neighbours what they had; ids outside the batch are reported
    lone = int(members[at[0], 3])
    members[at[0], 3] = -1
    keep = [i for i in range(q.shape[0]) if i != lone]
    out2 = ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, shared, grp[2], plan, out=torch.full_like(out, 3.0))
    assert torch.equal(out2[keep], out[keep]) and not bool(out2[lone].any())
    ops.check_device_errors()
    members[at[0], 3] = q.shape[0]
    out2 = ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, shared, grp[2], plan, out=torch.full_like(out, 3.0))
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    assert torch.equal(out2[keep], out[keep]) and not bool(out2[lone].any())
    # keys beyond the plan are left out and reported
    ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, (n, 64, 1, 192, 1))
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, (n, 192, 1, 64, 1))
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    # NaN in a member's own keys and values stays in that member's rows
    row, head, s, pages, st, end = parts[1]
    for cache in (1, 2):
        bad = [a.clone() if i == cache else a for i, a in enumerate(args)]
        bad[cache].view(torch.uint8)[pages[-1], hkv - 1, 5, 7] = 0x7F
        out3 = ops.paged_decode_attention_grouped_fp8(*bad, 0.1, *grp, plan)
        keep = [i for i in range(q.shape[0]) if i != row]
        assert torch.equal(out3[keep], out[keep]) and torch.equal(out3[row, :-(hq // hkv)], out[row, :-(hq // hkv)])
        assert bool(out3[row, -1].isnan().any())
    ops.check_device_errors()


def test_grouped_many_in_a_graph(cuda):
    """A captured call follows the group table, the lengths and the cache as they are when it is replayed, on a
    stream of its own."""
    g = gen(77)
    groups = many_groups(g, 40, 90, 100)
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, 16, 8, groups, cuda)
    n = q.shape[0]
    plan = ops.grouped_decode_plan_fp8(n, 40, 16, 8, 128, 128)
    assert ops._grouped_whole(16, 8, 40, *plan[1:])
    live = [t.clone() for t in args]
    members, shared, start = grp[0].clone(), grp[1].clone(), grp[2].clone()
    out = torch.empty_like(args[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_decode_attention_grouped_fp8(*live, 0.1, members, shared, start, plan, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_decode_attention_grouped_fp8(*live, 0.1, members, shared, start, plan, out=out)
        for shift in (0, 1, 7):  # groups elsewhere in the table, answers that have grown, other queries
            members.copy_(grp[0].roll(shift, 0))
            shared.copy_(grp[1].roll(shift, 0))
            live[6].copy_(torch.maximum(args[6] - shift, grp[2] - 1))
            live[0].copy_(args[0].roll(shift, 2))
            graph.replay()
            want = ops.paged_decode_attention_grouped_fp8(*live, 0.1, members, shared, start, plan)
            assert torch.equal(out, want)
    torch.cuda.current_stream().wait_stream(side)
    ops.check_device_errors()


def test_grouped_equals_plain_decode_where_nothing_is_skipped(cuda):
    """Prompts of whole pages: the shared and the unshared kernels attend the same keys; a sequence in no
    group gets zeros whatever the workspace holds, a member id outside the batch is reported."""
    g = gen(21)
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, 16, 8, [(256, [5, 70]), (512, [64])], cuda)
    plan = ops.grouped_decode_plan_fp8(3, 2, 16, 8, 512, 70)
    a = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan)
    b = ops.paged_decode_attention_fp8(*args, 0.1)
    assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=1e-2)
    members = grp[0].clone()
    lone = int(members[0, 1])
    members[0, 1] = -1
    out = torch.full_like(a, 3.0)
    keep = [i for i in range(3) if i != lone]
    ws = ops.workspace_fp8(3, 16, plan[2] + plan[4], cuda, grouped=True)
    for fill in (0, -1, 1, 5, 7 << 28):
        ws.view(torch.int32).fill_(fill)
        ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, *grp[1:], plan, out=out, workspace=ws)
        assert torch.equal(out[keep], a[keep]) and not bool(out[lone].any())
    ops.check_device_errors()
    members[0, 1] = 3
    ops.paged_decode_attention_grouped_fp8(*args, 0.1, members, *grp[1:], plan, out=out)
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    assert torch.equal(out[keep], a[keep])


# ------------------------------------------------------------------------------------------ prefill
PREFILL = [
    # hq, hkv, (cached tokens, new tokens)
    (16, 8, [(0, 1)]), (16, 8, [(0, 64), (0, 65), (0, 63)]), (16, 8, [(100, 1), (0, 200), (700, 130), (63, 1), (64, 2)]),
    (4, 2, [(300, 300), (0, 513)]), (8, 8, [(10, 100), (0, 7)]), (32, 8, [(5, 70), (250, 10)]),
    (40, 8, [(0, 90), (33, 33)]), (16, 1, [(70, 70), (1, 1)]), (32, 2, [(0, 130)]), (14, 2, [(128, 65)]),
]


@pytest.mark.parametrize("hq,hkv,seqs", PREFILL)
@pytest.mark.parametrize("tiled", [False, True])
def test_prefill(cuda, hq, hkv, seqs, tiled):
    g = gen(hq * 7 + len(seqs))
    lens = [p + n for p, n in seqs]
    nb = sum(-(-n // PAGE) for n in lens) + 1
    k, v, ks, vs = random_cache(g, nb, hkv)
    table = paged(g, lens, nb)
    spoil_dead(k, v, table, lens)
    nq = [n for _, n in seqs]
    cu_q = torch.tensor([0] + np.cumsum(nq).tolist(), dtype=torch.int32)
    cu_k = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32)
    T = sum(nq) + 3  # rows behind the last sequence
    q = torch.randn(T, hq, D, generator=g).to(BF)
    out = torch.full((T, hq, D), 5.0, dtype=BF, device=cuda)
    args = on(cuda, q, k, v, ks, vs, cu_q, cu_k)
    tiles = torch.from_numpy(ops.build_tiles(nq)).to(cuda) if tiled else None
    ops.attention_paged_prefill_fp8(*args, max(nq), table.to(cuda), 0.1, tiles=tiles, out=out)
    k64, v64 = values(k, ks), values(v, vs)
    for b, (past, n) in enumerate(seqs):
        rows = slice(int(cu_q[b]), int(cu_q[b + 1]))
        for h in range(hq):
            kv = [rows_of(c, table[b], 0, lens[b], h // (hq // hkv)) for c in (k64, v64)]
            check_attention(out[rows, h], *attend(q[rows, h], [kv], 0.1, past), f"sequence {b} head {h}")
    assert bool((out[sum(nq):] == 5.0).all())
    ops.check_device_errors()


@pytest.mark.parametrize("seqs", [[(0, 512)] * 8, [(3000, 300), (0, 1000), (511, 129)], [(0, 256), (0, 257), (4000, 256)] * 3])
def test_prefill_many_tiles(cuda, seqs):
    """Full waves of CTAs, tiles of all depths side by side, the call repeated back to back: no wait gives up."""
    g = gen(len(seqs))
    lens, nq = [p + n for p, n in seqs], [n for _, n in seqs]
    nb = sum(-(-n // PAGE) for n in lens)
    k, v, ks, vs = random_cache(g, nb, 8)
    table = paged(g, lens, nb)
    cu_q = torch.tensor([0] + np.cumsum(nq).tolist(), dtype=torch.int32)
    cu_k = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32)
    q = torch.randn(sum(nq), 16, D, generator=g).to(BF)
    args = on(cuda, q, k, v, ks, vs, cu_q, cu_k)
    outs = [ops.attention_paged_prefill_fp8(*args, max(nq), table.to(cuda), 0.1) for _ in range(12)]
    ops.check_device_errors()
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    k64, v64 = values(k, ks), values(v, vs)
    for b, (past, n) in enumerate(seqs):
        rows = slice(int(cu_q[b]), int(cu_q[b + 1]))
        for h in (b % 16, 15 - b):
            kv = [rows_of(c, table[b], 0, lens[b], h // 2) for c in (k64, v64)]
            check_attention(outs[0][rows, h], *attend(q[rows, h], [kv], 0.1, past), f"sequence {b} head {h}")


def test_prefill_nan_in_later_keys(cuda):
    """NaN in keys and values behind a row's last key, inside its own tile, stays out of the row; the rows
    that attend them are NaN."""
    g = gen(31)
    k, v, ks, vs = random_cache(g, 2, 2)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    for bad, cache in ((50, v), (50, k), (200, v), (299, v)):
        c = cache.clone()
        c.view(torch.uint8)[int(table[0, bad // PAGE]), 1, bad % PAGE, 5] = 0x7F
        kk, vv = (k, c) if cache is v else (c, v)
        q = torch.randn(300, 4, D, generator=g).to(BF)
        args = on(cuda, q, kk, vv, ks, vs, torch.tensor([0, 300], dtype=torch.int32),
                  torch.tensor([0, 300], dtype=torch.int32))
        out = ops.attention_paged_prefill_fp8(*args, 300, table.to(cuda), 0.1).cpu()
        k64, v64 = values(k, ks), values(v, vs)
        for h in range(4):
            kv = [rows_of(x, table[0], 0, 300, h // 2) for x in (k64, v64)]
            ref, mag, most = attend(q[:, h], [kv], 0.1, 0)
            upto = bad if h >= 2 else 300
            check_attention(out[:upto, h], ref[:upto], mag[:upto], most, f"key {bad} head {h}")
            if h >= 2:
                assert bool(out[bad:, h, 5].isnan().all())
        q1 = q[:1].to(cuda)  # the same for one token over the first keys
        dec = ops.paged_decode_attention_fp8(q1, *args[1:5], table.to(cuda), torch.tensor([bad], dtype=torch.int32,
                                             device=cuda), 0.1, seqlen_add=0)
        assert bool(torch.isfinite(dec).all())


@pytest.mark.parametrize("past,width", [(400, 1), (3000, 8)])
def test_prefill_keys_beyond_the_table_are_reported(cuda, past, width):
    """More keys than the table can name, in one split and in several: reported, and left out."""
    g = gen(33)
    k, v, ks, vs = random_cache(g, 9, 2)
    q = torch.randn(20, 4, D, generator=g).to(BF)
    table = torch.arange(1, width + 1, dtype=torch.int32)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    args = on(cuda, q, k, v, ks, vs, i32(0, 20), i32(0, 20 + past))
    n = ops.prefill_split_plan_fp8(1, 20, 20, 20 + past, 4, 2)[1]
    assert (n == 1) == (past == 400)
    out = ops.attention_paged_prefill_fp8(*args, 20, table.to(cuda), 0.1, max_seqlen_k=20 + past)
    with pytest.raises(ops.NativeError, match="page id"):
        ops.check_device_errors()
    k64, v64 = values(k, ks), values(v, vs)
    for h in range(4):
        kv = [rows_of(c, table[0], 0, width * PAGE, h // 2) for c in (k64, v64)]
        check_attention(out[:, h], *attend(q[:, h], [kv], 0.1, past))
    # a sequence of more queries than max_seqlen_q: the rows beyond are left, and reported
    q = torch.randn(300, 4, D, generator=g).to(BF)
    out = torch.full((300, 4, D), 2.0, dtype=BF, device=cuda)
    args = on(cuda, q, k, v, ks, vs, i32(0, 300), i32(0, 300))
    ops.attention_paged_prefill_fp8(*args, 100, torch.tensor([[1, 2]], dtype=torch.int32, device=cuda), 0.1, out=out)
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    assert bool((out[128:] == 2.0).all()) and not bool((out[:128] == 2.0).all())
    ops.check_device_errors()


def test_prefill_shapes_reported(cuda):
    """Fewer keys than queries, and a page outside the pool."""
    g = gen(32)
    k, v, ks, vs = random_cache(g, 3, 2)
    q = torch.randn(20, 4, D, generator=g).to(BF)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    out = torch.full((20, 4, D), 2.0, dtype=BF, device=cuda)
    args = on(cuda, q, k, v, ks, vs, i32(0, 20), i32(0, 10), torch.tensor([[0]], dtype=torch.int32))
    ops.attention_paged_prefill_fp8(*args[:7], 20, args[7], 0.1, out=out)
    with pytest.raises(ops.NativeError, match="inconsistent"):
        ops.check_device_errors()
    assert bool((out == 2.0).all())
    t = torch.tensor([[0, 3]], dtype=torch.int32, device=cuda)
    out = ops.attention_paged_prefill_fp8(*args[:6], i32(0, 300).to(cuda), 20, t, 0.1)
    with pytest.raises(ops.NativeError, match="page id"):
        ops.check_device_errors()
    k64, v64 = values(k, ks), values(v, vs)
    for h in range(4):
        kv = [rows_of(c, [0], 0, 256, h // 2) for c in (k64, v64)]
        check_attention(out[:, h], *attend(q[:, h], [kv], 0.1))


# ------------------------------------------------------------------------------------------ value scales
def leaning_cache(g, num_blocks, hkv, table, blocks, value_scale):
    """random_cache whose keys in the token blocks `blocks` of the sequence `table` score high where element 0
    of a query is positive and all others low; `value_scale`: of the blocks' values, by token block."""
    k, v, ks, vs = random_cache(g, num_blocks, hkv)
    ks[:] = 2.0 ** -6
    k[..., 0] = torch.tensor(-448.0).to(F8)
    for i in range(4 * len(table)):
        page, sub = int(table[i // 4]), i % 4
        vs[page, :, sub] = value_scale(i)
        if i in blocks:
            k[page, :, sub * BLOCK:(sub + 1) * BLOCK, 0] = torch.tensor(448.0).to(F8)
    return k, v, ks, vs


# The keys' lead is 2 * 0.1 * 7 * q0 (natural units): 2.02 bits of probability for each unit of q0.
VALUE_SCALES = [
    # blocks that lead, their lead in bits, exponents of the value scale of those blocks and of the others
    ([5], 161, -20, 0), ([5], 161, -24, 0), ([5], 161, -30, 0), ([5], 161, -60, 0), ([5], 161, -90, 0),
    ([0], 161, -30, 0), ([1, 3, 5, 7, 9], 161, -30, 0), ([1, 3, 5, 7, 9], 161, -60, 30), ([9], 60, -20, -4),
    # probabilities of 2^-30 and less that outweigh the others by their values
    ([0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11], 30, -30, 30), ([0, 2, 4, 6, 8, 10], 40, 0, 60), ([2], 40, 0, 40),
    ([4], 30, -126, 4), ([4], 100, -126, 100),
    # values near the end of the type's range
    ([3], 20, 119, 119), ([3], 20, -120, -120), ([3], 20, -60, 115),
]


def value_scale_case(lead, bits, small, other, rows=40, n=700):
    """(q, cache, table, per head the 64-bit keys and values) of one sequence whose last rows are queries."""
    g = gen(700 + bits + len(lead))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    cache = leaning_cache(g, 4, 2, table[0], lead, lambda i: 2.0 ** (small if i in lead else other))
    q = torch.randn(rows, 4, D, generator=g)
    q[:, :, 0] = bits / 2.02
    kv = [[rows_of(values(cache[i], cache[i + 2]), table[0], 0, n, h // 2) for i in (0, 1)] for h in range(4)]
    return q.to(BF), cache, table, kv


def zero_block_cases():
    """Blocks whose values are all zero, under the smallest scale and under a scale of zero."""
    for zero in (2.0 ** -126, 0.0):
        for blocks, big in (([0, 1, 6], 0), ([1, 3, 5, 7, 9], 110), (list(range(10)), -20)):
            q, (k, v, ks, vs), table, _ = value_scale_case(blocks, 0, 0, big)
            for i in blocks:
                v.view(torch.uint8)[int(table[0, i // 4]), :, i % 4 * 64:i % 4 * 64 + 64] = 0
                vs[int(table[0, i // 4]), :, i % 4] = zero
            kv = [[rows_of(values(*c), table[0], 0, 700, h // 2) for c in ((k, ks), (v, vs))] for h in range(4)]
            yield q, (k, v, ks, vs), table, kv, f"zeros under {zero} in {blocks}:"


def check_prefill_values(dev, q, cache, table, kv, msg=""):
    """A sequence whose last rows are queries: many copies side by side take one split, one with room for
    more keys in its table takes several."""
    rows, n = q.shape[0], kv[0][0].shape[0]
    args = on(dev, *cache)
    for copies, width in ((64, 3), (1, 24)):
        assert (ops.prefill_split_plan_fp8(copies, copies * rows, rows, width * PAGE, 4, 2)[1] > 1) == (copies == 1)
        cu_q, cu_k = (torch.arange(copies + 1, dtype=torch.int32, device=dev) * i for i in (rows, n))
        t = torch.cat([table, torch.full((1, width - 3), -1, dtype=torch.int32)], 1).to(dev).repeat(copies, 1)
        out = ops.attention_paged_prefill_fp8(q.to(dev).repeat(copies, 1, 1), *args, cu_q, cu_k, rows, t, 0.1)
        assert torch.equal(out[:rows], out[-rows:])
        for h in range(4):
            check_attention(out[:rows, h], *attend(q[:, h], [kv[h]], 0.1, n - rows), f"{msg} {copies} copies, head {h}")
    ops.check_device_errors()


@pytest.mark.parametrize("lead,bits,small,other", VALUE_SCALES)
def test_prefill_weighs_value_scales_with_the_probabilities(cuda, lead, bits, small, other):
    """Blocks of values whose scales are far apart, where the probabilities and not the scales alone say which
    of them an output is made of.  What is rounded to halves is a probability weighed by its block's scale
    against a reference that follows the largest of those, so the bound is that of any other call."""
    check_prefill_values(cuda, *value_scale_case(lead, bits, small, other))


def test_prefill_value_blocks_of_zeros_take_their_probability(cuda):
    for q, cache, table, kv, msg in zero_block_cases():
        check_prefill_values(cuda, q, cache, table, kv, msg)


def check_decode_values(dev, q, cache, table, kv, msg=""):
    """A sequence's last token: plain and grouped (512 keys shared), in one split and in several."""
    n = kv[0][0].shape[0]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = on(dev, q[-1:], *cache, table)
    outs = [ops.paged_decode_attention_fp8(*args, i32(n - 1), 0.1, **kw)
            for kw in ({}, {"split_tokens": 128, "max_splits": 6}, {"split_tokens": 64, "max_splits": 11})]
    for plan in ((32, 512, 1, 192, 1), (1, 192, 3, 64, 3)):  # a CTA for all keys, and splits
        members = torch.full((32, 8), -1, dtype=torch.int32, device=dev)
        members[3, 0] = 0
        shared = torch.zeros(32, dtype=torch.int32, device=dev)
        shared[3] = 512
        outs.append(ops.paged_decode_attention_grouped_fp8(*args, i32(n - 1), 0.1, members, shared, i32(512), plan))
    assert ops._grouped_whole(4, 2, 32, 512, 1, 192, 1)
    for h in range(4):
        ref = attend(q[-1:, h], [kv[h]], 0.1)
        for i, out in enumerate(outs):
            check_attention(out[:, h], *ref, f"{msg} call {i} head {h}")
    ops.check_device_errors()


@pytest.mark.parametrize("lead,bits,small,other", VALUE_SCALES)
def test_decode_weighs_value_scales_with_the_probabilities(cuda, lead, bits, small, other):
    check_decode_values(cuda, *value_scale_case(lead, bits, small, other))


def test_decode_value_blocks_of_zeros_take_their_probability(cuda):
    for q, cache, table, kv, msg in zero_block_cases():
        check_decode_values(cuda, q, cache, table, kv, msg)


def test_a_zeroed_cache_gives_zeros(cuda):
    """Scales of zero everywhere, as a cache is made: every form writes zeros."""
    k, v, ks, vs = ops.kv_cache_fp8(3, 2, cuda)
    q = torch.randn(20, 4, D, generator=gen(726)).to(BF).to(cuda)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table, out = i32(2, 0, 1).view(1, 3), torch.full((1, 4, D), 3.0, dtype=BF, device=cuda)
    members, shared = i32(0, *[-1] * 255).view(32, 8), i32(512, *[0] * 31)
    calls = [lambda kw=kw: ops.paged_decode_attention_fp8(q[:1], k, v, ks, vs, table, i32(699), 0.1, out=out, **kw)
             for kw in ({}, {"split_tokens": 128, "max_splits": 6})]
    calls += [lambda plan=plan: ops.paged_decode_attention_grouped_fp8(q[:1], k, v, ks, vs, table, i32(699), 0.1, members,
                                                                       shared, i32(512), plan, out=out)
              for plan in ((32, 512, 1, 192, 1), (1, 192, 3, 64, 3))]
    for i, call in enumerate(calls):
        out.fill_(3.0)
        assert not bool(call().any()), f"call {i}"
    for t in (table, torch.cat([table, i32(*[-1] * 21).view(1, 21)], 1)):
        assert not bool(ops.attention_paged_prefill_fp8(q, k, v, ks, vs, i32(0, 20), i32(0, 700), 20, t, 0.1,
                                                        out=torch.full_like(q, 3.0)).any())
    ops.check_device_errors()


@pytest.mark.parametrize("plan", [(10, 192, 1, 192, 1), (10, 64, 3, 64, 3)])
def test_grouped_value_scales_far_apart_in_some_groups(cuda, plan):
    """CTAs that take several groups one after another, some of them with value scales far apart: those follow the
    formula, the others keep their bits."""
    g = gen(725)
    groups = many_groups(g, 40, 150, 140)
    q, k, v, ks, vs, parts, args, grp = grouped_inputs(g, 16, 8, groups, cuda)
    assert ops._grouped_whole(16, 8, *plan) == (plan[1] == 192)
    before = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan)
    far, row = set(), 0
    for i, (_, own) in enumerate(groups):
        if i in (1, 5, 11, 12, 38):
            far |= {parts[row + j][0] for j in range(len(own))}
            for _, head, _, pages, _, _ in parts[row:row + len(own)]:
                for page in {*head, *pages}:
                    vs[page] = torch.exp2(torch.randint(-40, 40, vs[page].shape, generator=g).float())
        row += len(own)
    args[4] = vs.to(cuda)
    out = ops.paged_decode_attention_grouped_fp8(*args, 0.1, *grp, plan)
    near = [i for i in range(q.shape[0]) if i not in far]
    assert torch.equal(out[near], before[near])
    k64, v64 = values(k, ks), values(v, vs)
    for r, head, s, pages, a, b in parts:
        for h in (0, 7, 15) if r in far else ():
            kv = [torch.cat([rows_of(c, head, 0, s, h // 2), rows_of(c, pages, a, b, h // 2)]) for c in (k64, v64)]
            check_attention(out[r, h:h + 1], *attend(q[r, h:h + 1], [kv], 0.1), f"row {r} head {h}")
    ops.check_device_errors()


# ------------------------------------------------------------------------------------------ rows and elements
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (8, 8), (32, 2), (40, 8)])
def test_prefill_rows_without_a_tile_are_left(cuda, hq, hkv, listed):
    """Queries beyond max_seqlen_q, or of no listed tile, are left as they were where the keys are split too,
    whatever the workspace held; the others are right."""
    g = gen(730 + hq)
    seqs = [(2000, 300), (2500, 10), (1700, 200)] if hkv == 2 else [(3000, 300 if hq == 8 else 130)]
    lens, nq = [p + n for p, n in seqs], [n for _, n in seqs]
    nb = sum(-(-n // PAGE) for n in lens)
    k, v, ks, vs = random_cache(g, nb, hkv)
    table = paged(g, lens, nb, width=16)
    cu_q, cu_k = ([0] + np.cumsum(x).tolist() for x in (nq, lens))
    q = torch.randn(cu_q[-1], hq, D, generator=g).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    unit = max(64, 16 << max(i for i in range(5) if (16 << i) * (hq // hkv) <= 256))  # rows of a CTA's tile, or 64
    if listed:  # all but the second tile of each sequence
        tiles = torch.from_numpy(ops.build_tiles(nq)).view(-1, 2)
        tiles = tiles[(tiles[:, 1] < unit) | (tiles[:, 1] >= 2 * unit)].contiguous().to(cuda)
        left = lambda i: unit <= i < 2 * unit  # noqa: E731
    else:
        tiles = None
        left = lambda i: i >= unit  # noqa: E731
    max_q = max(nq) if listed else unit
    assert ops.prefill_split_plan_fp8(len(seqs), cu_q[-1], max_q, 16 * PAGE, hq, hkv)[1] > 1
    junk = [torch.full((1 << 24,), math.nan, device=cuda) for _ in range(2)]  # what a workspace may find
    del junk
    out = torch.full((cu_q[-1], hq, D), 2.0, dtype=BF, device=cuda)
    ops.attention_paged_prefill_fp8(*on(cuda, q, k, v, ks, vs), i32(cu_q), i32(cu_k), max_q, table.to(cuda), 0.1, tiles=tiles,
                                    out=out)
    if listed or max(nq) <= unit:
        ops.check_device_errors()
    else:
        with pytest.raises(ops.NativeError, match="inconsistent"):
            ops.check_device_errors()
    k64, v64 = values(k, ks), values(v, vs)
    for b, (past, n) in enumerate(seqs):
        rest = torch.tensor([left(i) for i in range(n)])
        rows = out[cu_q[b]:cu_q[b + 1]].cpu()
        assert bool((rows[rest] == 2.0).all()), f"sequence {b}"
        for h in (0, hq - 1):
            kv = [rows_of(c, table[b], 0, lens[b], h // (hq // hkv)) for c in (k64, v64)]
            ref, mag, most = attend(q[cu_q[b]:cu_q[b + 1], h], [kv], 0.1, past)
            check_attention(rows[~rest, h], ref[~rest], mag[~rest], most, f"sequence {b} head {h}")


def check_with_nan(out, q, k, v, scale, past=None, msg=""):
    """Element d of a row is NaN exactly where a key that the row attends has NaN in element d of its value."""
    at = ~torch.isfinite(v)
    ref, mag, most = attend(q, [[k, torch.where(at, 0.0, v)]], scale, past)
    sees = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool)
    if past is not None:
        sees = torch.arange(k.shape[0]) <= past + torch.arange(q.shape[0])[:, None]
    want = (sees.double() @ at.double()) > 0
    out = out.cpu()
    assert torch.equal(out.isnan(), want), f"{msg} NaN in {int(out.isnan().sum())} elements, not {int(want.sum())}"
    check_attention(torch.where(want, torch.zeros_like(out), out), torch.where(want, 0.0, ref), mag, most, msg)


@pytest.mark.parametrize("hq,hkv", [(4, 2), (8, 8), (32, 2), (5, 1)])
@pytest.mark.parametrize("past", [0, 90, 1500])
def test_nan_values_reach_their_element_of_the_rows_that_attend_them(cuda, hq, hkv, past):
    """Whatever the tile that holds them -- one that every row sees, or one that some rows see in part --
    and in decode as in prefill, in one split and in several."""
    g = gen(740 + hq + past)
    n = 300
    nb = -(-(past + n) // PAGE)
    k, v, ks, vs = random_cache(g, nb, hkv)
    table = paged(g, [past + n], nb)
    for _ in range(14):
        key, h = int(torch.randint(0, past + n, (1,), generator=g)), int(torch.randint(0, hkv, (1,), generator=g))
        e = torch.randint(0, D, (2,), generator=g)
        v.view(torch.uint8)[int(table[0, key // PAGE]), h, key % PAGE, e] = torch.tensor([0x7F, 0xFF], dtype=torch.uint8)
    q = torch.randn(n, hq, D, generator=g).to(BF)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    args = on(cuda, q, k, v, ks, vs)
    k64, v64 = values(k, ks), values(v, vs)
    wide = torch.full((1, 64), -1, dtype=torch.int32)
    wide[:, :nb] = table
    outs = [ops.attention_paged_prefill_fp8(*args, i32(0, n), i32(0, past + n), n, t.to(cuda), 0.1) for t in (table, wide)]
    at = [0, 63, 64, 150, n - 1]
    dec = [ops.paged_decode_attention_fp8(args[0][at], *args[1:], table.to(cuda).expand(len(at), -1), i32(*[past + i for i in at]),
                                          0.1, **kw) for kw in ({}, {"split_tokens": 128, "max_splits": 15})]
    for h in range(hq):
        kv = [rows_of(c, table[0], 0, past + n, h // (hq // hkv)) for c in (k64, v64)]
        for out in outs:
            check_with_nan(out[:, h], q[:, h], *kv, 0.1, past, f"prefill head {h}")
        for out in dec:
            for r, i in enumerate(at):
                check_with_nan(out[r:r + 1, h], q[i:i + 1, h], *[c[:past + i + 1] for c in kv], 0.1, None, f"decode {i} head {h}")
    ops.check_device_errors()


def test_infinite_queries_give_nan(cuda):
    """A head whose query holds an infinity: some score is +inf, the softmax has no value, all of the head's
    outputs are NaN; the other heads and rows are as before.  One split and several."""
    g = gen(750)
    k, v, ks, vs = random_cache(g, 3, 2)
    table = torch.tensor([[1, 0, 2]], dtype=torch.int32)
    q = torch.randn(3, 4, D, generator=g).to(BF)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    args = on(cuda, k, v, ks, vs)
    wide = torch.cat([table, torch.full((1, 29), -1, dtype=torch.int32)], 1).to(cuda)
    calls = [lambda x: ops.paged_decode_attention_fp8(x, *args, table.to(cuda).expand(3, -1), i32(600, 99, 700), 0.1),
             lambda x: ops.paged_decode_attention_fp8(x, *args, table.to(cuda).expand(3, -1), i32(600, 99, 700), 0.1,
                                                      split_tokens=64, max_splits=12),
             lambda x: ops.attention_paged_prefill_fp8(x, *args, i32(0, 3), i32(0, 700), 3, table.to(cuda), 0.1),
             lambda x: ops.attention_paged_prefill_fp8(x, *args, i32(0, 3), i32(0, 700), 3, wide, 0.1)]
    for value in (math.inf, -math.inf):
        bad = q.clone()
        bad[1, 3, 0] = value
        for i, call in enumerate(calls):
            a, b = call(q.to(cuda)), call(bad.to(cuda))
            assert bool(b[1, 3].isnan().all()), f"call {i}"
            assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, :3], b[1, :3]), f"call {i}"
    ops.check_device_errors()


# ------------------------------------------------------------------------------------------ store
def scale_for(top):
    if top == 0:
        return 2.0 ** -126
    m, e = math.frexp(top)
    return 2.0 ** max(-126, e - 9 if m <= 0.875 else e - 8)


def ref_rows(qkv, pos, cs, qw, kw, hq, hkv, eps=1e-6):
    x = qkv.double().view(-1, hq + 2 * hkv, D)
    w = torch.cat([qw.double().expand(hq, D), kw.double().expand(hkv, D)])
    y = x[:, :hq + hkv]
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w
    c, s = cs[pos][:, None, :64].double(), cs[pos][:, None, 64:].double()
    lo, hi = y[..., :64], y[..., 64:]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    return y[:, :hq], y[:, hq:], x[:, hq + hkv:]


def check_store(before, after, new, slots):
    """codes and scales of K or V after a store of rows `new` [T, hkv, 128] (64 bits) at `slots`."""
    (c0, s0), (c1, s1) = before, after
    last = {}
    for t, s in enumerate(slots):
        if 0 <= s < c0.shape[0] * PAGE:
            last[s] = t
    blocks = {}
    for s, t in last.items():
        blocks.setdefault(s // BLOCK, []).append((s % BLOCK, t))
    same = torch.ones(c0.shape[0] * 4, dtype=torch.bool)
    for blk, rows in blocks.items():
        same[blk] = False
        page, sub = blk // 4, blk % 4
        for h in range(c0.shape[1]):
            x = torch.stack([new[t, h] for _, t in rows])
            top = x[torch.isfinite(x)].abs().max().item() if torch.isfinite(x).any() else 0.0
            anew = any(r == 0 for r, _ in rows)
            was, now = s0[page, h, sub].item(), s1[page, h, sub].item()
            need = {scale_for(top * (1 + 2.0 ** -18)), scale_for(top * (1 - 2.0 ** -18))}
            assert now in ({n if anew else max(n, was) for n in need}), (blk, h, now, need, was)
            old, got = c0[page, h].view(4, BLOCK, D)[sub], c1[page, h].view(4, BLOCK, D)[sub]
            here = torch.zeros(BLOCK, dtype=torch.bool)
            here[[r for r, _ in rows]] = True
            keep = old if anew or now <= was else (old.float() * (was / now)).to(F8)
            assert torch.equal(keep[~here].view(torch.uint8), got[~here].view(torch.uint8)), (blk, h)
            for r, t in rows:
                want, code = new[t, h] / now, got[r].double()
                fine = torch.isfinite(want)
                assert bool(code[~fine].isnan().all())
                want, code = want[fine], code[fine]
                step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -6))) - 3)
                near = want.abs().max().item() * 2.0 ** -18 if len(want) else 0.0
                assert bool(((code - want).abs() <= step / 2 + near).all()), (blk, h, r)
    u0, u1 = c0.view(torch.uint8), c1.view(torch.uint8)
    b0 = u0.reshape(c0.shape[0], c0.shape[1], 4, -1).transpose(1, 2).reshape(len(same), -1)
    b1 = u1.reshape(c0.shape[0], c0.shape[1], 4, -1).transpose(1, 2).reshape(len(same), -1)
    assert torch.equal(b0[same], b1[same])
    assert torch.equal(s0.transpose(1, 2).reshape(len(same), -1)[same], s1.transpose(1, 2).reshape(len(same), -1)[same])


def run_store(dev, g, hq, hkv, slots, num_blocks, gain=None, wide=0, positions=None, qkv=None):
    T = len(slots)
    k, v, ks, vs = random_cache(g, num_blocks, hkv)
    if qkv is None:
        qkv = torch.randn(T, hq + 2 * hkv, D, generator=g)
        if gain is not None:
            qkv = qkv * gain[:, None, None]
        qkv = qkv.view(T, -1).to(BF)
    qw = (1 + 0.3 * torch.randn(D, generator=g)).to(BF)
    kw = (1 + 0.3 * torch.randn(D, generator=g)).to(BF)
    cs = torch.randn(512, D, generator=g)
    pos = torch.randint(0, 512, (T,), generator=g) if positions is None else positions
    big = torch.zeros(T, qkv.shape[1] + wide, dtype=BF)
    big[:, :qkv.shape[1]] = qkv
    dk, dv, dks, dvs = on(dev, k, v, ks, vs)
    qkv_d = big.to(dev)[:, :qkv.shape[1]]
    q = ops.qk_norm_rope_store_fp8(qkv_d, *on(dev, pos, cs, qw, kw), 1e-6, hq, hkv, dk, dv, dks, dvs,
                                   torch.tensor(slots, dtype=torch.int32, device=dev))
    rq, rk, rv = ref_rows(qkv, pos, cs, qw, kw, hq, hkv)
    near = rq.abs().amax(-1, keepdim=True) * 2.0 ** -18
    ok = torch.isfinite(rq)
    assert bool(((q.double().cpu() - rq).abs() <= rq.abs() * 2.0 ** -8 + near)[ok].all())
    check_store((k, ks), (dk.cpu(), dks.cpu()), rk, slots)
    check_store((v, vs), (dv.cpu(), dvs.cpu()), rv, slots)
    return dk, dv, dks, dvs


def chunk(page, a, b):
    return [page * PAGE + j for j in range(a, b)]


STORE = [
    # hq, hkv, slots, pages
    (16, 8, [700], 4), (16, 8, [64 * i + (i % 64) for i in range(16)], 4), (4, 2, chunk(1, 0, 256), 3),
    (16, 8, chunk(0, 5, 70) + chunk(2, 0, 1) + chunk(1, 255, 256) + chunk(1, 100, 200), 3),
    (40, 8, chunk(0, 3, 5), 1), (2, 1, [-1, 3, -1, 130, -1], 1), (14, 2, chunk(0, 0, 256) + chunk(1, 0, 200), 2),
    # tokens of a block apart from one another, out of order, the same slot twice and three times
    (4, 2, [5, 300, 6, 301, 4, 200, 7], 2), (4, 2, [63, 1, 62, 2, 0, 40], 1), (4, 2, [9, 9], 1),
    (4, 2, [130, 5, 130, 6, 130, 7, 8, 9, 10, 11, 12, 130], 1), (4, 2, [10] + [64 + i for i in range(20)] + [10, 11], 1),
    (4, 2, [300 + 64 * (i % 3) for i in range(30)], 3),
]


@pytest.mark.parametrize("hq,hkv,slots,nb", STORE)
@pytest.mark.parametrize("wide", [0, 40])
def test_store(cuda, hq, hkv, slots, nb, wide):
    g = gen(len(slots) + hq)
    gain = torch.exp(2 * torch.randn(len(slots), generator=g))  # V values over several scales
    run_store(cuda, g, hq, hkv, slots, nb, gain=gain, wide=wide)
    ops.check_device_errors()


def test_store_many_tokens(cuda):
    """More tokens than a scan covers at once, in runs of all lengths."""
    g = gen(77)
    slots, nb = [], 40
    for p in torch.randperm(nb, generator=g).tolist():
        a = int(torch.randint(0, 200, (1,), generator=g))
        slots += chunk(p, a, min(256, a + int(torch.randint(1, 250, (1,), generator=g))))
    run_store(cuda, g, 4, 2, slots, nb)
    ops.check_device_errors()


def test_store_values_that_are_not_finite(cuda):
    """Infinities and NaN become NaN codes and leave the scale alone; zeros take the smallest scale; the
    largest and the smallest bf16 values keep theirs."""
    g = gen(78)
    hq, hkv, T = 2, 1, 70
    x = torch.randn(T, 4, D, generator=g)
    x[3, 3, 7], x[4, 3, 9], x[5, 3, 1] = math.inf, -math.inf, math.nan
    x[6, 3] = 0
    run_store(cuda, g, hq, hkv, chunk(0, 0, T), 1, qkv=x.view(T, -1).to(BF))
    for fill in (0.0, 3.3895e38, 1e-38):
        y = torch.randn(3, 4, D, generator=g)
        y[:, 3] = fill
        run_store(cuda, g, hq, hkv, [64, 65, 66], 1, qkv=y.view(3, -1).to(BF))
    ops.check_device_errors()


def test_store_in_any_chunks(cuda):
    """A block filled token by token holds the scale of one filled at once, and its codes but for those
    that a raised scale pushed into the subnormals (rounded twice)."""
    g = gen(79)
    T, hq, hkv = 150, 4, 2
    qkv = (torch.randn(T, 8, D, generator=g) * torch.exp(torch.randn(T, 1, 1, generator=g))).view(T, -1).to(BF)
    cs, w = torch.randn(T, D, generator=g), torch.ones(D, dtype=BF)
    args = on(cuda, qkv, torch.arange(T), cs, w)
    slots = torch.arange(T, dtype=torch.int32, device=cuda)
    caches = []
    for step in (T, 1, 7, 64):
        c = ops.kv_cache_fp8(1, hkv, cuda)
        for x in c[:2]:
            x.view(torch.uint8).fill_(0x55)  # a recycled page
        for x in c[2:]:
            x.fill_(1e9)
        for a in range(0, T, step):
            s = slice(a, min(T, a + step))
            ops.qk_norm_rope_store_fp8(args[0][s], args[1][s], args[2], args[3], args[3], 1e-6, hq, hkv, *c, slots[s])
        caches.append([x.cpu() for x in c])
    for c in caches[1:]:
        assert torch.equal(c[2][:, :, :3], caches[0][2][:, :, :3]) and torch.equal(c[3][:, :, :3], caches[0][3][:, :, :3])
        for i in (0, 1):
            a, b = caches[0][i][:, :, :T].float(), c[i][:, :, :T].float()
            assert bool(((a - b).abs() <= 2.0 ** -9).all()), "codes differ beyond one subnormal step"
            assert bool((a == b)[b.abs() > 2.0 ** -6].all())


def test_store_reports_and_skips(cuda):
    """Slots outside the pool are reported and skipped, positions outside the table are reported."""
    g = gen(80)
    run_store(cuda, g, 4, 2, [5, 2 * PAGE, 7, -2, 1 << 30], 2)
    with pytest.raises(ops.NativeError, match="slot"):
        ops.check_device_errors()
    ops.check_device_errors()
    k, v, ks, vs = on(cuda, *random_cache(g, 1, 1))
    qkv = torch.randn(2, 4 * D, generator=g).to(BF).to(cuda)
    w = torch.ones(D, dtype=BF, device=cuda)
    ops.qk_norm_rope_store_fp8(qkv, torch.tensor([3, 99], device=cuda), torch.zeros(8, D, device=cuda), w, w, 1e-6, 2, 1,
                               k, v, ks, vs, torch.tensor([0, 1], dtype=torch.int32, device=cuda))
    with pytest.raises(ops.NativeError, match="positions"):
        ops.check_device_errors()


# ------------------------------------------------------------------------------------------ together
def test_store_then_attend_in_a_graph_on_a_side_stream(cuda):
    """Prompt, then decode steps replayed as one CUDA graph (store + decode), twice over two workspaces
    captured apart, against the 64-bit attention of what the cache holds."""
    g = gen(90)
    hq, hkv, nb, P = 16, 8, 6, 130
    cache = ops.kv_cache_fp8(nb, hkv, cuda)
    cs = torch.randn(400, D, generator=g)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(BF)
    cs_d, w_d = on(cuda, cs, w)
    table = torch.tensor([[4, 1], [2, 5]], dtype=torch.int32)
    table_d = table.to(cuda)

    def tokens(n):
        return torch.randn(n, (hq + 2 * hkv) * D, generator=g).to(BF)

    pos = torch.arange(P).repeat(2)
    slots = torch.cat([table[b, torch.arange(P) // PAGE] * PAGE + torch.arange(P) % PAGE for b in range(2)]).int()
    q = ops.qk_norm_rope_store_fp8(tokens(2 * P).to(cuda), pos.to(cuda), cs_d, w_d, w_d, 1e-6, hq, hkv, *cache, slots.to(cuda))
    cu = torch.tensor([0, P, 2 * P], dtype=torch.int32, device=cuda)
    out = ops.attention_paged_prefill_fp8(q, *cache, cu, cu, P, table_d, 0.1)
    k64, v64 = values(cache[0].cpu(), cache[2].cpu()), values(cache[1].cpu(), cache[3].cpu())
    for b in range(2):
        for h in (0, 7, 15):
            kv = [rows_of(c, table[b], 0, P, h // 2) for c in (k64, v64)]
            rows = slice(b * P, (b + 1) * P)
            check_attention(out[rows, h], *attend(q[rows, h].cpu(), [kv], 0.1, 0))

    side = torch.cuda.Stream()
    qkv_s, pos_s = torch.zeros(2, (hq + 2 * hkv) * D, dtype=BF, device=cuda), torch.zeros(2, dtype=torch.long, device=cuda)
    slot_s, ctx_s = torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    plan = ops.decode_split_plan_fp8(2, hkv, 2 * PAGE)
    graphs = []
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        slot_s.fill_(-1)
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                qs = ops.qk_norm_rope_store_fp8(qkv_s, pos_s, cs_d, w_d, w_d, 1e-6, hq, hkv, *cache, slot_s)
                o = ops.paged_decode_attention_fp8(qs, *cache, table_d, ctx_s, 0.1, split_tokens=plan[0], max_splits=plan[1])
            graphs.append((gr, qs, o))
        for i in range(140):
            at = P + i
            qkv_s.copy_(tokens(2).to(cuda))
            pos_s.fill_(at)
            ctx_s.fill_(at)
            slot_s.copy_(torch.tensor([int(table[b, at // PAGE]) * PAGE + at % PAGE for b in range(2)], dtype=torch.int32))
            gr, qs, o = graphs[i % 2]
            gr.replay()
            if i in (0, 1, 61, 62, 125, 126, 127, 139):
                side.synchronize()
                k64, v64 = values(cache[0].cpu(), cache[2].cpu()), values(cache[1].cpu(), cache[3].cpu())
                for b in range(2):
                    for h in (0, 9):
                        kv = [rows_of(c, table[b], 0, at + 1, h // 2) for c in (k64, v64)]
                        check_attention(o[b, h:h + 1], *attend(qs[b, h:h + 1].cpu(), [kv], 0.1), f"step {i}")
    torch.cuda.default_stream().wait_stream(side)
    del graphs
    ops.check_device_errors()


def test_pages_beyond_32_bit_offsets(cuda):
    """A pool of more than 2^32 bytes of codes: the last page is read and written where it lies."""
    hkv, nb = 8, 16500  # 262144 bytes a page: 4.3e9
    k, v, ks, vs = ops.kv_cache_fp8(nb, hkv, cuda)
    g = gen(91)
    last = nb - 1
    qkv = torch.randn(70, 32 * D, generator=g).to(BF)
    cs, w = torch.randn(70, D, generator=g), torch.ones(D, dtype=BF)
    slots = torch.arange(70, dtype=torch.int32) + last * PAGE
    q = ops.qk_norm_rope_store_fp8(*on(cuda, qkv, torch.arange(70), cs, w, w), 1e-6, 16, hkv, k, v, ks, vs, slots.to(cuda))
    _, rk, rv = ref_rows(qkv, torch.arange(70), cs, w, w, 16, hkv)
    k64, v64 = values(k[last:].cpu(), ks[last:].cpu()), values(v[last:].cpu(), vs[last:].cpu())
    assert bool(((k64[0, :, :70].transpose(0, 1) - rk).abs() <= 2.0 ** -4 * rk.abs() + rk.abs().max() * 2.0 ** -15).all())
    table = torch.tensor([[last]], dtype=torch.int32, device=cuda)
    dec = ops.paged_decode_attention_fp8(q[69:], k, v, ks, vs, table, torch.tensor([69], dtype=torch.int32, device=cuda), 0.1)
    cu = torch.tensor([0, 70], dtype=torch.int32, device=cuda)
    pre = ops.attention_paged_prefill_fp8(q, k, v, ks, vs, cu, cu, 70, table, 0.1)
    for h in range(16):
        kv = [c[0, h // 2, :70] for c in (k64, v64)]
        check_attention(dec[:, h], *attend(q[69:, h].cpu(), [kv], 0.1))
        check_attention(pre[:, h], *attend(q[:, h].cpu(), [kv], 0.1, 0))
    assert not bool(k[:last].view(torch.uint8).any())
    ops.check_device_errors()


def test_refusals(cuda):
    """Calls that the kernels cannot take raise before anything runs."""
    k, v, ks, vs = ops.kv_cache_fp8(2, 2, cuda)
    q = torch.zeros(1, 4, D, dtype=BF, device=cuda)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    t, n = i32(0).view(1, 1), i32(5)
    dec = ops.paged_decode_attention_fp8
    bad = [
        lambda: dec(q.float(), k, v, ks, vs, t, n, 0.1),
        lambda: dec(q[:, :3], k, v, ks, vs, t, n, 0.1),
        lambda: dec(q.expand(1, 4, D).repeat(1, 9, 1), k, v, ks, vs, t, n, 0.1),  # 18 query heads a kv head
        lambda: dec(q, k.view(torch.uint8), v, ks, vs, t, n, 0.1),
        lambda: dec(q, k, v[:1], ks, vs, t, n, 0.1),
        lambda: dec(q, k, v, ks[:, :, :3], vs, t, n, 0.1),
        lambda: dec(q, k[:, :, :128], v[:, :, :128], ks, vs, t, n, 0.1),
        lambda: dec(q, k, v, ks, vs, t.long(), n, 0.1),
        lambda: dec(q, k, v, ks, vs, t, n.long(), 0.1),
        lambda: dec(q, k, v, ks, vs, t, i32(5, 6), 0.1),
        lambda: dec(q, k, v, ks, vs, t, n, 0.1, split_tokens=100, max_splits=3),
        lambda: dec(q, k, v, ks, vs, t, n, 0.1, split_tokens=128),
        lambda: dec(q, k, v, ks, vs, t, n, 0.1, split_tokens=16384, max_splits=1),
        lambda: dec(q, k, v, ks, vs, t, n, 0.1, split_tokens=64, max_splits=4, workspace=torch.zeros(8, device=cuda)),
        lambda: dec(q, k, v, ks, vs, t, n.cpu(), 0.1),
        lambda: dec(q, k, v, ks, vs, t, n, 0.1, out=torch.zeros(1, 4, D, device=cuda)),
        lambda: ops.qk_norm_rope_store_fp8(torch.zeros(1, 5 * D, dtype=BF, device=cuda), n.long(), torch.zeros(8, D, device=cuda),
                                           q[0, 0], q[0, 0], 1e-6, 4, 2, k, v, ks, vs, n),
        lambda: ops.attention_paged_prefill_fp8(q, k, v, ks, vs, i32(0, 1), i32(0, 1, 2), 1, t, 0.1),
        lambda: ops.paged_decode_attention_grouped_fp8(q, k, v, ks, vs, t, n, 0.1, i32(0, -1).view(1, 2), i32(3), i32(0), (1, 64, 1, 64, 1)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ops.NativeError):
            f()
            pytest.fail(f"call {i} was taken")
    # no groups: no sequence is in one
    z = ops.paged_decode_attention_grouped_fp8(q, k, v, ks, vs, t, n, 0.1, t[:0, :1].expand(0, 8).contiguous(), n[:0], n,
                                               ops.grouped_decode_plan_fp8(q.shape[0], 0, 4, 2, 0, 64))
    assert z.shape == q.shape and not bool(z.any())
    # tensors of another device than the current one (as seen where the current one is asked for)
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(torch.cuda, "current_device", lambda: 1)
        with pytest.raises(ops.NativeError, match="current CUDA device"):
            dec(q, k, v, ks, vs, t, n, 0.1)
    # nothing to do is taken: no rows, no tokens
    e = torch.empty(0, 4, D, dtype=BF, device=cuda)
    assert dec(e, k, v, ks, vs, t[:0], n[:0], 0.1, max_ctx=1).shape == (0, 4, D)
    r = ops.qk_norm_rope_store_fp8(torch.zeros(0, 8 * D, dtype=BF, device=cuda), n[:0].long(), torch.zeros(8, D, device=cuda),
                                   q[0, 0], q[0, 0], 1e-6, 4, 2, k, v, ks, vs, n[:0])
    assert r.shape == (0, 4, D)
    assert ops.attention_paged_prefill_fp8(e, k, v, ks, vs, i32(0, 0), i32(0, 0), 0, t, 0.1).shape == (0, 4, D)
    ops.check_device_errors()
