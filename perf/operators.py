"""Measured cases of the 8-bit paged KV cache: the store that fills it and the three attentions that read it.

The cache holds e4m3 codes, ``k_cache`` and ``v_cache`` [num_blocks, kv_heads, 256, 128], and one fp32
scale for every block of 64 tokens and head, ``k_scale`` and ``v_scale`` [num_blocks, kv_heads, 4]: a
stored value is code * scale.  The operators:

  store    QK-norm and rotation of a projected token row; the rotated queries are returned, keys and
           values are appended to the cache.  A block's scale is the smallest power of two under which
           everything appended to it since its first row stays within 448; where a later token raises
           it, the rows already there are rounded again under the new scale.
  decode   attention of one query token per sequence over its pages.
  grouped  the same where up to eight sequences share their first keys.
  prefill  causal attention of a chunk of query tokens per sequence over its pages.
"""
import math

import torch

own = False

D = 128        # head width
PAGE = 256     # tokens of a page
BLOCK = 64     # tokens that share a scale
TOP = 448.0    # largest e4m3 value
EPS = 1e-6
MAX_POS = 40960
DEV = "cuda"


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the chat user's next token: one row through the store, launch latency counts
        {"name": "store one token", "op": "store", "kind": "decode", "n": 1, "top": 700, "hq": 16, "hkv": 8},
        # a rollout's decode step: 64 prompts x 8 completions, each row at its own place of its own block
        {"name": "store 512 rows", "op": "store", "kind": "decode", "n": 512, "top": 1024, "hq": 16, "hkv": 8},
        # prompts of a rollout entering the cache together, chunks that begin and end inside blocks
        {"name": "store 37 chunks", "op": "store", "kind": "chunk", "n": 37, "top": 512, "hq": 16, "hkv": 8},
        # one chat user in the middle of an answer
        {"name": "decode one sequence", "op": "decode", "n": 1, "top": 700, "hq": 16, "hkv": 8},
        # a rollout's decode step without shared prompts
        {"name": "decode 512 sequences", "op": "decode", "n": 512, "top": 1024, "hq": 16, "hkv": 8},
        # a few users with long documents
        {"name": "decode 16 long", "op": "decode", "n": 16, "top": 32768, "hq": 16, "hkv": 8},
        # wider head groups, odd lengths
        {"name": "decode wide groups", "op": "decode", "n": 33, "top": 5000, "hq": 32, "hkv": 4},
        # a small rollout: groups of different sizes
        {"name": "grouped 5 groups", "op": "grouped", "n": 5, "members": 0, "shared": 300, "top": 130, "hq": 16, "hkv": 8},
        # the middle of the default rollout: 64 prompts x 8 completions, 256 answered tokens
        {"name": "grouped 64 groups", "op": "grouped", "n": 64, "members": 8, "shared": 512, "top": 512, "hq": 16, "hkv": 8},
        # several short prompts and single tokens in one mixed step
        {"name": "prefill short ragged", "op": "prefill", "n": 11, "q": 90, "past": 400, "hq": 16, "hkv": 8},
        # fresh prompts of one scheduler step
        {"name": "prefill fresh prompts", "op": "prefill", "n": 8, "q": 512, "past": 0, "hq": 16, "hkv": 8},
        # a chunk of 2048 tokens far into a long document
        {"name": "prefill long chunk", "op": "prefill", "n": 1, "q": 2048, "past": 30720, "hq": 16, "hkv": 8},
    ]


HEADS = [(16, 8), (16, 8), (16, 8), (4, 2), (32, 8), (8, 8), (40, 8), (32, 4), (16, 2), (16, 1)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "decode", "grouped", "prefill"])
    hq, hkv = rng.choice(HEADS)
    if op == "store":
        kind = rng.choice(["decode", "chunk"])
        n = _log(rng, 1, 512) if kind == "decode" else _log(rng, 1, 32)
        return {"op": op, "kind": kind, "n": n, "top": _log(rng, 16, 1024 if kind == "decode" else 400), "hq": hq, "hkv": min(hkv, 8)}
    if op == "decode":
        top = _log(rng, 8, 32768)
        return {"op": op, "n": _log(rng, 1, max(1, min(512, 300000 // top))), "top": top, "hq": hq, "hkv": hkv}
    if op == "grouped":
        return {"op": op, "n": _log(rng, 1, 48), "members": rng.randrange(0, 9), "shared": _log(rng, 8, 700), "top": _log(rng, 4, 500), "hq": hq, "hkv": hkv}
    past = rng.choice([0, _log(rng, 16, 8192)])
    q = _log(rng, 2, 1024)
    return {"op": op, "n": _log(rng, 1, max(1, min(24, 4000 // q))), "q": q, "past": past, "hq": min(hq, 16), "hkv": min(hkv, 8)}


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Per sequence (tokens already cached, new tokens): the case's own, whatever the seed."""
    host = torch.Generator().manual_seed(case["n"] + case["hq"])
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=host))  # noqa: E731
    op, n = case["op"], case["n"]
    if op == "store" and case["kind"] == "decode" or op == "decode":
        lo = max(0, case["top"] // 16 if n > 1 else case["top"] - case["top"] // 8)
        return [(pick(lo, case["top"]) - 1 if case["top"] > 0 else 0, 1) for _ in range(n)]
    if op == "store":
        past = [pick(0, 3) * 37 if i % 3 == 1 else 0 for i in range(n)]
        return [(p, pick(max(1, case["top"] // 8), case["top"])) for p in past]
    if n == 1:
        return [(case["past"], case["q"])]
    return [(pick(0, case["past"]), 1 if case["past"] and i % 4 == 3 else pick(max(1, case["q"] // 2), case["q"])) for i in range(n)]


def _codes(gen, num_blocks, hkv):
    """Cache contents as a running program holds them: codes that use their block's range, scales of
    neighbouring powers of two."""
    codes = torch.empty(num_blocks, hkv, PAGE, D, dtype=torch.float8_e4m3fn, device=DEV)
    for a in range(0, num_blocks, 512):
        b = min(num_blocks, a + 512)
        x = torch.randn(b - a, hkv, PAGE, D, generator=gen, dtype=torch.bfloat16, device=DEV)
        codes[a:b] = (x * 100).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)
    e = torch.randint(-7, -3, (num_blocks, hkv, PAGE // BLOCK), generator=gen, device=DEV)
    return codes, torch.exp2(e.float())


def _tables(totals, host, spare=3):
    """Page tables of sequences with `totals` tokens over a pool in random order: int32 rows padded with -1."""
    pages = [-(-t // PAGE) for t in totals]
    pool = torch.randperm(sum(pages) + spare, generator=host, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(totals), max(1, max(pages))), -1, dtype=torch.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = pool[at:at + p]
        at += p
    return table, sum(pages) + spare


def _int(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).to(DEV)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv, op = case["hq"], case["hkv"], case["op"]
    s = {"op": op, "hq": hq, "hkv": hkv, "scale": D ** -0.5}
    if op == "grouped":
        return _prepare_grouped(case, s, host, gen)
    lens = _lengths(case)
    table, num_blocks = _tables([p + n for p, n in lens], host)
    s["k_cache"], s["k_scale"] = _codes(gen, num_blocks, hkv)
    s["v_cache"], s["v_scale"] = _codes(gen, num_blocks, hkv)
    if op == "store":
        pos = torch.cat([torch.arange(p, p + n) for p, n in lens])
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor([n for _, n in lens]))
        s["slots"] = (table[seq, pos // PAGE].long() * PAGE + pos % PAGE).to(torch.int32).to(DEV)
        s["positions"] = pos.to(DEV)
        T = pos.numel()
        x = torch.randn(T, hq + 2 * hkv, D, generator=gen, device=DEV)
        s["qkv"] = (x * torch.exp(0.5 * torch.randn(T, 1, 1, generator=gen, device=DEV))).reshape(T, -1).to(torch.bfloat16)
        w = 1 + 0.2 * torch.randn(2, D, generator=gen, device=DEV)
        w[:, ::37] *= 4  # a few loud channels, as trained norms have
        s["q_norm"], s["k_norm"] = w[0].to(torch.bfloat16), w[1].to(torch.bfloat16)
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float) / D))
        ang = torch.outer(torch.arange(MAX_POS, dtype=torch.float), inv)
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=-1).to(DEV)
        return s
    s["table"] = table.to(DEV)
    if op == "decode":
        s["seqlens"] = _int([p for p, _ in lens])
        s["max_ctx"] = max(p for p, _ in lens) + 1
        s["q"] = torch.randn(len(lens), hq, D, generator=gen, device=DEV).to(torch.bfloat16)
        return s
    nq, nk = [n for _, n in lens], [p + n for p, n in lens]
    s["cu_q"] = _int([0] + torch.tensor(nq).cumsum(0).tolist())
    s["cu_k"] = _int([0] + torch.tensor(nk).cumsum(0).tolist())
    s["max_q"], s["max_k"] = max(nq), max(nk)
    s["q"] = torch.randn(sum(nq), hq, D, generator=gen, device=DEV).to(torch.bfloat16)
    return s


def _groups(case):
    """Per group (members, shared keys), and per member its own keys: the case's own, whatever the seed."""
    host = torch.Generator().manual_seed(case["n"] + case["hq"])
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=host))  # noqa: E731
    size = [case["members"] or 1 + i % 8 for i in range(case["n"])]
    shared = [pick(max(1, case["shared"] // 8), case["shared"]) for _ in size]
    own_keys = [[pick(max(1, case["top"] // 3), case["top"]) for _ in range(m)] for m in size]
    return size, shared, own_keys


def _prepare_grouped(case, s, host, gen):
    size, shared, own_keys = _groups(case)
    n = sum(size)
    start = [-(-p // PAGE) * PAGE for p in shared]  # own keys begin on a page of their own
    need = sum(-(-p // PAGE) for p in shared) + sum(-(-k // PAGE) for row in own_keys for k in row) + 3
    pool = torch.randperm(need, generator=host).tolist()
    width = max(st // PAGE + max(-(-k // PAGE) for k in row) for st, row in zip(start, own_keys))
    table = torch.full((n, width), -1, dtype=torch.int32)
    members = torch.full((case["n"], 8), -1, dtype=torch.int32)
    lens, first, b = [], [], 0
    for g, (m, st, row) in enumerate(zip(size, start, own_keys)):
        head = [pool.pop() for _ in range(st // PAGE)]
        for j, k in enumerate(row):
            pages = head + [pool.pop() for _ in range(-(-k // PAGE))]
            table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            members[g, j] = b
            lens.append(st + k - 1)
            first.append(st)
            b += 1
    s["k_cache"], s["k_scale"] = _codes(gen, need, case["hkv"])
    s["v_cache"], s["v_scale"] = _codes(gen, need, case["hkv"])
    s["table"], s["members"] = table.to(DEV), members.to(DEV)
    s["seqlens"], s["kv_start"], s["shared_len"] = _int(lens), _int(first), _int(shared)
    s["group_of"] = torch.repeat_interleave(torch.arange(case["n"]), torch.tensor(size)).to(DEV)
    s["max_shared"], s["max_own"] = max(shared), max(max(r) for r in own_keys)
    s["q"] = torch.randn(n, case["hq"], D, generator=gen, device=DEV).to(torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from qwen3_naive_inference_b200 import ops
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["op"] == "store":
        q = ops.qk_norm_rope_store_fp8(s["qkv"], s["positions"], s["cos_sin"], s["q_norm"], s["k_norm"], EPS, s["hq"], s["hkv"], *cache, s["slots"])
        return (q, *cache)
    if s["op"] == "decode":
        return ops.paged_decode_attention_fp8(s["q"], *cache, s["table"], s["seqlens"], s["scale"], max_ctx=s["max_ctx"])
    if s["op"] == "grouped":
        plan = ops.grouped_decode_plan_fp8(s["q"].shape[0], s["members"].shape[0], s["hq"], s["hkv"], s["max_shared"], s["max_own"])
        return ops.paged_decode_attention_grouped_fp8(s["q"], *cache, s["table"], s["seqlens"], s["scale"], s["members"], s["shared_len"], s["kv_start"], plan)
    return ops.attention_paged_prefill_fp8(s["q"], *cache, s["cu_q"], s["cu_k"], s["max_q"], s["table"], s["scale"])


def _run_plain(s):
    if s["op"] == "store":
        return _plain_store(s)
    if s["op"] == "decode":
        lens = s["seqlens"] + 1
        at = torch.arange(s["max_ctx"], device=DEV).expand(lens.numel(), -1)
        return _plain_rows(s, s["table"], at, at < lens[:, None])
    if s["op"] == "grouped":
        # key j of a row: one of the group's shared keys, or the row's own key j - shared_len
        shared = s["shared_len"][s["group_of"]][:, None]
        j = torch.arange(s["max_shared"] + s["max_own"], device=DEV)[None]
        at = torch.where(j < shared, j, s["kv_start"][:, None] + j - shared)
        owner = s["members"][s["group_of"], 0].long()  # shared keys: the first member's pages
        page = torch.where(j < shared, _page(s["table"][owner], at), _page(s["table"], at))
        return _plain_rows(s, page, at, at < (s["seqlens"] + 1)[:, None], paged=True)
    return _plain_prefill(s)


def _page(table, at):
    return table.gather(1, (at // PAGE).clamp(0, table.shape[1] - 1))


def _values(codes, scales, page, at):
    """fp32 keys or values at positions `at` [n, L] of rows with pages `page` [n, L]: [n, heads, L, D]."""
    x = codes[page, :, at % PAGE].float() * scales[page, :, at % PAGE // BLOCK].unsqueeze(-1)
    return x.transpose(1, 2)


def _softmax(x):
    """Softmax over the last axis in 32 bits; a row with nothing but -inf gives zeros."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_rows(s, table, at, seen, paged=False):
    """One query row per sequence over the keys at `at` that `seen` allows."""
    page = (table if paged else _page(table, at)).clamp_min(0).long()
    k, v = _values(s["k_cache"], s["k_scale"], page, at), _values(s["v_cache"], s["v_scale"], page, at)
    q = s["q"].float().view(-1, s["hkv"], s["hq"] // s["hkv"], D)
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    p = _softmax(score.masked_fill(~seen[:, None, None], -math.inf))
    return (p @ v).reshape(s["q"].shape).to(torch.bfloat16)


def _plain_prefill(s):
    nq, nk = s["cu_q"].diff(), s["cu_k"].diff()
    i, j = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    row = (s["cu_q"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1)  # padded: [batch, max_q]
    q = s["q"].float()[row].transpose(1, 2)
    at = j.expand(nq.numel(), -1)
    page = _page(s["table"], at).clamp_min(0).long()
    group = s["hq"] // s["hkv"]
    k = _values(s["k_cache"], s["k_scale"], page, at)
    v = _values(s["v_cache"], s["v_scale"], page, at)
    q = q.reshape(nq.numel(), s["hkv"], group * s["max_q"], D)
    seen = (j <= (nk - nq)[:, None, None] + i[:, None]) & (j < nk[:, None, None])  # [batch, max_q, max_k]
    score = ((q @ k.transpose(-1, -2)) * s["scale"]).view(nq.numel(), s["hkv"], group, s["max_q"], s["max_k"])
    p = _softmax(score.masked_fill(~seen[:, None, None], -math.inf)).view(nq.numel(), s["hkv"], group * s["max_q"], s["max_k"])
    o = (p @ v).view(nq.numel(), s["hq"], s["max_q"], D).transpose(1, 2)
    return o[i < nq[:, None]].to(torch.bfloat16)


def _plain_store(s):
    hq, hkv = s["hq"], s["hkv"]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, D)
    w = torch.cat([s["q_norm"].float().expand(hq, D), s["k_norm"].float().expand(hkv, D)])
    y = x[:, :hq + hkv]
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
    cs = s["cos_sin"][s["positions"]][:, None]
    c, sn, lo, hi = cs[..., :D // 2], cs[..., D // 2:], y[..., :D // 2], y[..., D // 2:]
    y = torch.cat([lo * c - hi * sn, hi * c + lo * sn], dim=-1)
    _plain_append(s["k_cache"], s["k_scale"], y[:, hq:], s["slots"].long())
    _plain_append(s["v_cache"], s["v_scale"], x[:, hq + hkv:], s["slots"].long())
    return y[:, :hq].to(torch.bfloat16), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_append(codes, scales, x, slots):
    page, sub, row = slots // PAGE, slots % PAGE // BLOCK, slots % PAGE
    old = scales.clone()
    old[page[row % BLOCK == 0], :, sub[row % BLOCK == 0]] = 0  # first row written: the block begins anew
    top = torch.zeros_like(scales).transpose(1, 2).reshape(-1, scales.shape[1])
    top.scatter_reduce_(0, (slots // BLOCK)[:, None].expand(-1, scales.shape[1]), x.abs().amax(-1), "amax")
    m, e = torch.frexp(top)  # top = m 2^e with m in [1/2, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).masked_fill(top == 0, -126).clamp_min(-126)
    need = torch.ldexp(torch.ones_like(top), e).view(-1, PAGE // BLOCK, scales.shape[1]).transpose(1, 2)
    hit = torch.zeros_like(scales, dtype=torch.bool)
    hit[page, :, sub] = True
    new = torch.where(hit, torch.maximum(old, need), old)
    grown = hit & (old > 0) & (new > old)
    blocks = codes.view(*scales.shape, BLOCK, D)
    blocks[grown] = (blocks[grown].float() * (old[grown] / new[grown])[:, None, None]).to(codes.dtype)
    codes[page, :, row] = (x / new[page, :, sub].unsqueeze(-1)).to(codes.dtype)
    scales.copy_(new)


# ---------------------------------------------------------------------------------------------- floors
def work(case):
    """Each input read once, each output written once."""
    hq, hkv, op = case["hq"], case["hkv"], case["op"]
    row = 2 * hkv * (D + 4 / BLOCK)  # bytes of one token's codes and its share of the scales
    if op == "grouped":
        size, shared, own_keys = _groups(case)
        keys = sum(shared) + sum(map(sum, own_keys))
        pairs = sum(m * p for m, p in zip(size, shared)) + sum(map(sum, own_keys))
        return {"bytes": keys * row + sum(size) * hq * D * 4, "flops": 4 * hq * D * pairs}
    lens = _lengths(case)
    T = sum(n for _, n in lens)
    if op == "store":
        return {"bytes": T * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + row + D * 4 + 12), "flops": T * (hq + hkv) * D * 8}
    keys = sum(p + n for p, n in lens)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens)
    return {"bytes": keys * row + T * hq * D * 4, "flops": 4 * hq * D * pairs}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "store":
        return _exact_store(s)
    k64 = lambda pages, h, n: _exact_kv(s["k_cache"], s["k_scale"], pages, h, n)  # noqa: E731
    v64 = lambda pages, h, n: _exact_kv(s["v_cache"], s["v_scale"], pages, h, n)  # noqa: E731
    group = s["hq"] // s["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    table = s["table"].cpu()

    def attend(rows, parts, past):
        """Rows of one sequence over the keys of `parts` [(pages, first, last)]; row i sees past + i + 1 of them."""
        for h in range(s["hkv"]):
            k = torch.cat([k64(p, h, b)[a:] for p, a, b in parts])
            v = torch.cat([v64(p, h, b)[a:] for p, a, b in parts])
            q = s["q"][rows, h * group:(h + 1) * group].double()
            x = torch.einsum("igd,jd->gij", q, k) * s["scale"]
            if q.shape[0] > 1:
                i, j = torch.arange(q.shape[0], device=DEV)[:, None], torch.arange(k.shape[0], device=DEV)
                x = x.masked_fill(j > past + i, -math.inf)
            out[rows, h * group:(h + 1) * group] = torch.einsum("gij,jd->igd", torch.softmax(x, -1), v)

    if s["op"] == "prefill":
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for b in range(len(cq) - 1):
            nk, nq = ck[b + 1] - ck[b], cq[b + 1] - cq[b]
            attend(slice(cq[b], cq[b + 1]), [(table[b], 0, nk)], nk - nq)
    elif s["op"] == "decode":
        for b, n in enumerate(s["seqlens"].tolist()):
            if n >= 0:
                attend(slice(b, b + 1), [(table[b], 0, n + 1)], n)
    else:
        lens, first, shared = s["seqlens"].tolist(), s["kv_start"].tolist(), s["shared_len"].tolist()
        for g, members in enumerate(s["members"].tolist()):
            for b in [m for m in members if m >= 0]:
                attend(slice(b, b + 1), [(table[members[0]], 0, shared[g]), (table[b], first[b], lens[b] + 1)], 0)
    return out


def _exact_kv(codes, scales, pages, h, n):
    pages = pages[:-(-n // PAGE)].long().to(DEV)
    x = codes[pages, h].double().view(-1, PAGE // BLOCK, BLOCK, D) * scales[pages, h].double()[:, :, None, None]
    return x.reshape(-1, D)[:n]


def _exact_round(x):
    """Nearest e4m3 value (ties to the even code) of 64-bit numbers within +-448."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -30)))
    e = torch.where(torch.exp2(e) > x.abs(), e - 1, torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, e))
    step = torch.exp2(e.clamp_min(-6) - 3)
    return torch.round(x / step) * step


def _exact_store(s):
    hq, hkv = s["hq"], s["hkv"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    z = torch.view_as_complex(s["cos_sin"][s["positions"]].double().view(-1, 2, D // 2).transpose(1, 2).contiguous())

    def turn(y, w):
        y = y / (y.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        r = torch.complex(y[..., :D // 2], y[..., D // 2:]) * z[:, None]
        return torch.cat([r.real, r.imag], -1)

    q, k, v = turn(x[:, :hq], s["q_norm"]), turn(x[:, hq:hq + hkv], s["k_norm"]), x[:, hq + hkv:]
    slots = s["slots"].cpu().long()
    order = torch.argsort(slots // BLOCK, stable=True)
    blocks, count = torch.unique_consecutive(slots[order] // BLOCK, return_counts=True)
    got = {}
    for name, y in (("k", k), ("v", v)):
        codes, scales = s[name + "_cache"].double(), s[name + "_scale"].double()
        at = 0
        for blk, c in zip(blocks.tolist(), count.tolist()):
            mine = order[at:at + c]
            at += c
            page, sub, rows = blk // 4, blk % 4, (slots[mine] % PAGE).to(DEV)
            new = y[mine.to(DEV)]
            most = new.abs().amax((0, 2)) / TOP
            up = torch.ceil(torch.log2(most.clamp_min(2.0 ** -126)))
            up = torch.where(torch.exp2(up - 1) >= most, up - 1, torch.where(torch.exp2(up) < most, up + 1, up))  # log2 may be an ulp off
            need = torch.exp2(up.clamp_min(-126))
            if int(slots[mine].min()) % BLOCK:
                was = scales[page, :, sub]
                need = torch.maximum(was, need)
                part = codes[page, :, sub * BLOCK:(sub + 1) * BLOCK]
                part.copy_(torch.where((need > was)[:, None, None], _exact_round(part * (was / need)[:, None, None]), part))
            scales[page, :, sub] = need
            codes[page][:, rows] = _exact_round((new / need[None, :, None]).transpose(0, 1))
        got[name] = codes, scales
    return q, got["k"][0], got["v"][0], got["k"][1], got["v"][1]
