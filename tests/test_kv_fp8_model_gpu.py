"""The model on the 8-bit paged KV cache (``kv_cache_dtype = "fp8"``): every paged path -- prefill in one
and in many chunks, eager and captured decode steps, the grouped rollout, the whole GRPO step -- runs on it.

The cache's contents are taken as they are (their own error is tested with the kernels), so the checks of
values hold the model against attention over the codes the model stored; the rest is equality.
"""
import math

import pytest
import torch

from qwen3_naive_inference_b200 import ops
from qwen3_naive_inference_b200 import qwen3_grpo_train as G
from qwen3_naive_inference_b200.qwen3_naive import BlockManager, Qwen3Config, Sequence, build_model

pytestmark = pytest.mark.gpu

TINY = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=256,
            num_hidden_layers=2, vocab_size=512, max_position_embeddings=4096)


@pytest.fixture(scope="module")
def model(cuda):
    m = build_model(Qwen3Config(**TINY), device=cuda, seed=3, std=0.05)
    m._num_blocks = 48
    m.kv_cache_dtype = "fp8"
    return m


def prompts(cuda, lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (1, n), generator=g).to(cuda) for n in lens]


def prefill(model, seq, n):
    seq.num_scheduled_tokens = n
    ids, pos, cu_q, cu_k, mq, mk, blk, bt = model._prepare_step([seq])
    with torch.no_grad():
        h = model.model.forward_prefill(ids, pos, cu_q, cu_k, mq, mk, blk, bt)
    seq.kv_len += n
    return h


def test_cache_layout_and_size(model):
    half = model._block_bytes()
    model.allocate_global_kv_cache()
    a = model.model.layers[1].self_attn
    assert a.k_cache.dtype == torch.float8_e4m3fn and a.k_cache.shape == (48, 2, 256, 128)
    assert a.k_scale.shape == (48, 2, 4) and a.k_cache.is_contiguous() and a.v_scale.is_contiguous()
    model.kv_cache_dtype = "bf16"
    try:
        assert half * 2 == model._block_bytes() + 2 * 2 * 2 * 2 * 4 * 4  # and the scales
        model.kv_cache_dtype = "int3"
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            model.allocate_global_kv_cache()
    finally:
        model.kv_cache_dtype = "fp8"


def test_layer_attends_to_what_it_stored(model, cuda):
    """A layer's paged prefill against attention in 64 bits over the codes and scales it left in the cache.
    The projection, the query's rounding and o_proj are bf16: errors of a few 2^-8 of the largest output."""
    model.allocate_global_kv_cache()
    at = model.model.layers[0].self_attn
    T = 300
    x = torch.randn(T, 256, device=cuda, generator=torch.Generator(device=cuda).manual_seed(5)).to(torch.bfloat16)
    pos = torch.arange(T, device=cuda)
    table = torch.tensor([[7, 3]], dtype=torch.int32, device=cuda)
    slots = (table[0].long()[pos // 256] * 256 + pos % 256).int()
    cu = torch.tensor([0, T], dtype=torch.int32, device=cuda)
    with torch.no_grad():
        got = at.forward_prefill(x, pos, cu, cu, T, T, slots, table)
        qkv = ops.linear(x, at.qkv_proj.weight)
        q = ops.qk_norm_rope(qkv, pos, at._cos_sin(cuda), at.q_norm.weight, at.k_norm.weight, at.eps, 4, 2)
    q = q[:, :512].double().view(T, 4, 128)

    def values(c, s):
        v = c.double().view(48, 2, 4, 64, 128) * s.double()[..., None, None]
        return v.view(48, 2, 256, 128)[table[0].long()].transpose(0, 1).reshape(2, 512, 128)[:, :T]

    k, v = values(at.k_cache, at.k_scale), values(at.v_cache, at.v_scale)
    raw = qkv[:, 768:].double().view(T, 2, 128).transpose(0, 1)
    assert (v - raw).abs().max() <= 2.0 ** -4 * raw.abs().max()
    s = torch.einsum("ihd,hjd->hij", q, k.repeat_interleave(2, 0)) * at.scale
    s = s.masked_fill(torch.ones(T, T, device=cuda, dtype=torch.bool).triu(1), -math.inf)
    o = torch.einsum("hij,hjd->ihd", torch.softmax(s, -1), v.repeat_interleave(2, 0)).reshape(T, 512)
    ref = o @ at.o_proj.weight.double().T
    assert (got.double() - ref).abs().max() <= 4 * 2.0 ** -8 * ref.abs().max()
    ops.check_device_errors()


def test_chunked_prefill_stores_the_same_cache(model):
    """One chunk and many: the same scales, the same codes but where a later chunk raised a scale."""
    model.allocate_global_kv_cache()
    toks = torch.randint(0, 512, (700,), generator=torch.Generator().manual_seed(4)).tolist()
    at = model.model.layers[0].self_attn
    left = []
    for sizes in ([700], [256, 256, 188], [1, 99, 100, 250, 250]):
        seq = Sequence(toks)
        BlockManager(model._num_blocks, 256).allocate(seq)
        for n in sizes:
            h = prefill(model, seq, n)
        page = seq.block_table[1]
        left.append((at.k_cache[page].float(), at.v_cache[page].float(), at.k_scale[page].clone(), at.v_scale[page].clone(), h[-1].float()))
    for k, v, ks, vs, last in left[1:]:
        assert torch.equal(ks, left[0][2]) and torch.equal(vs, left[0][3])
        assert (k - left[0][0]).abs().max() <= 2.0 ** -9 and (v - left[0][1]).abs().max() <= 2.0 ** -9
        assert (last - left[0][4]).abs().max() <= 0.05 * left[0][4].abs().max()
    ops.check_device_errors()


def test_generation_reads_only_written_cache_slots(model, cuda):
    """NaN codes and NaN scales in every page beforehand change no token, in any paged path."""
    ps = prompts(cuda, (3, 250, 256, 300, 17), seed=13)
    model.allocate_global_kv_cache()

    def run(code, scale):
        for layer in model.model.layers:
            at = layer.self_attn
            for c in (at.k_cache, at.v_cache):
                c.view(torch.uint8).fill_(code)
            for s in (at.k_scale, at.v_scale):
                s.fill_(scale)
        model._has_cuda_graphs = False  # recapture: the capture warm-up runs on this pool too
        out = []
        for graphs in (True, False):
            model.use_cuda_graphs = graphs
            torch.manual_seed(0)
            out.append(model.generate_continuous(ps, max_new_tokens=20, top_k=1, temperature=1.0)[1])
            torch.manual_seed(0)
            out.append(model.generate_grouped_with_logprobs(ps[:3], 3, max_new_tokens=20, top_k=1, temperature=1.0)[1])
        model.use_cuda_graphs = True
        out.append(model.generate_kvcache(ps[1], max_new_tokens=8, top_k=1, temperature=1.0).tolist())
        return out

    zero = run(0, 0.0)
    assert run(0x7F, math.nan) == zero
    assert run(0x55, 3.0e38) == zero
    ops.check_device_errors()


def test_formats_change_over(model, cuda):
    """bf16 and 8-bit caches in turn: each gives what it gave before."""
    ps = prompts(cuda, (40, 300, 9), seed=2)

    def run():
        torch.manual_seed(0)
        return model.generate_continuous_with_logprobs(ps, max_new_tokens=12, top_k=1, temperature=1.0)

    first = run()
    model.kv_cache_dtype = "bf16"
    try:
        wide = run()
    finally:
        model.kv_cache_dtype = "fp8"
    assert model.model.layers[0].self_attn.k_scale is None
    again = run()
    assert again[0] == first[0] and again[2] == first[2]
    assert [len(t) for t in wide[0]] == [len(t) for t in first[0]]


def test_grpo_step_on_the_8_bit_cache(model, cuda):
    """The whole step: rollout on the 8-bit cache, log-probs, loss and update on the model itself.  The
    rollout's log-probs are those of the policy but for the cache's rounding."""
    opt = torch.optim.SGD(model.parameters(), lr=0.0)
    torch.manual_seed(0)
    out = G.grpo_step(model, opt, prompts(cuda, (70, 200), seed=8), group_size=4, max_new_tokens=40, temperature=1.0,
                      rewards=torch.arange(8).float(), beta=0.0, return_batch=True)
    assert out["completion_tokens"] == 320 and math.isfinite(out["loss"])
    b = out["batch"]
    now = G.batch_log_probs(model, b)
    off = ((now - b.old_lp) * b.mask).abs()
    # every key's score and every value within 2^-4 of itself: log-probs of a flat 512-way softmax move little
    assert off.max() < 0.5 and off.sum() / b.mask.sum() < 0.05
    ops.check_device_errors()
