"""Host side of the 8-bit paged KV cache (CPU only): argument checks of the entry points, split plans."""
import ctypes

import pytest
import torch

from qwen3_naive_inference_b200 import _lib, ops

A = ctypes.c_void_p(1 << 20)  # an aligned address that is never read: every call below is refused on the host
ODD = ctypes.c_void_p((1 << 20) + 8)


def decode(lib, q=A, q_stride=2048, k=A, ks=A, bt=A, seqlens=A, batch=1, hq=16, hkv=8, D=128, page=256, split=64, n=1, ws=None,
           out=A, pages=4, width=1):
    return lib.qb_paged_decode_attn_fp8(q, q_stride, k, A, ks, A, pages, page, bt, 1, width, seqlens, 1, batch, hq, hkv, D, 1.0,
                                        split, n, ws, out, None, None)


def test_decode_refusals():
    lib = _lib.load()
    assert decode(lib, D=64) == 2 and decode(lib, page=128) == 2
    for kw in ({"q": None}, {"q": ODD}, {"k": None}, {"k": ODD}, {"ks": None}, {"bt": None}, {"seqlens": None}, {"out": None},
               {"batch": -1}, {"hq": 15}, {"hq": 136}, {"hkv": 0}, {"hq": 0}, {"split": 0}, {"split": 96}, {"split": 8256},
               {"n": 0}, {"n": 2}, {"q_stride": 2044}, {"q_stride": 1024}, {"pages": -1}, {"pages": 1 << 24}, {"width": -1}):
        assert decode(lib, **kw) == 1, kw
    assert decode(lib, batch=0) == 0


def test_grouped_refusals():
    lib = _lib.load()

    def call(ws=A, members=A, n_groups=1, shared=(64, 1), own=(64, 1), D=128, step=1):
        return lib.qb_paged_decode_attn_grouped_fp8(A, 2048, A, A, A, A, 4, 256, A, 1, 1, A, 1, 1, 16, 8, D, 1.0, members, A,
                                                    n_groups, A, step, *shared, *own, ws, A, None, None)

    assert call(D=96) == 2
    assert call(step=0) == 1 and call(ws=None) == 1 and call(members=None) == 1 and call(n_groups=-1) == 1
    assert call(shared=(100, 1)) == 1 and call(own=(64, 0)) == 1 and call(own=(16384, 1)) == 1
    assert call(n_groups=0) == 0


def test_prefill_refusals():
    lib = _lib.load()

    def call(q=A, cu=A, batch=1, total=4, o_stride=2048, n_tiles=0, tps=1, page=256, hq=16, split=(0, 1), ws=None):
        return lib.qb_attn_paged_prefill_fp8(q, 2048, A, A, A, A, 4, page, A, 1, 1, cu, A, batch, None, n_tiles, tps, hq, 8, 128,
                                             1.0, *split, ws, A, o_stride, total, None, None)

    assert call(page=64) == 2
    for kw in ({"q": None}, {"cu": None}, {"batch": -1}, {"total": -1}, {"o_stride": 2044}, {"o_stride": 8}, {"tps": -1},
               {"n_tiles": -1}, {"hq": 17}, {"total": 1 << 31}, {"split": (128, 0)}, {"split": (128, 2)}, {"split": (64, 2), "ws": A},
               {"split": (0, 2), "ws": A}, {"split": (128, 70000), "ws": A}):
        assert call(**kw) == 1, kw
    assert call(batch=0) == 0 and call(total=0) == 0


def test_store_refusals():
    lib = _lib.load()

    def call(qkv=A, T=1, ld=4096, hq=16, hkv=8, D=128, pos=A, cs=A, max_pos=8, slots=A, pages=4, page=256, q=A, k=A, ks=A):
        return lib.qb_qk_norm_rope_store_fp8(qkv, T, ld, hq, hkv, D, pos, cs, max_pos, A, A, 1e-6, q, k, A, ks, A, slots, pages,
                                             page, None, None)

    assert call(D=64) == 2 and call(page=16) == 2
    for kw in ({"qkv": None}, {"qkv": ODD}, {"T": -1}, {"ld": 4088}, {"ld": 4100}, {"hq": 0}, {"hkv": 0}, {"pos": None},
               {"cs": ODD}, {"max_pos": 0}, {"slots": None}, {"pages": 1 << 23}, {"q": None}, {"k": ODD}, {"ks": None},
               {"T": 1 << 31}):
        assert call(**kw) == 1, kw
    assert call(T=0) == 0


def test_workspace_size():
    lib = _lib.load()
    assert lib.qb_paged_decode_fp8_workspace_bytes(4, 16, 1) == 0
    assert lib.qb_paged_decode_fp8_workspace_bytes(4, 16, 3) == 4 * 16 * 3 * 132 * 4
    assert lib.qb_paged_decode_fp8_workspace_bytes(4096, 128, 512) == 4096 * 128 * 512 * 132 * 4  # past 32 bits
    assert lib.qb_attn_paged_prefill_fp8_workspace_bytes(10, 16, 1) == 0
    assert lib.qb_attn_paged_prefill_fp8_workspace_bytes(1 << 20, 16, 64) == (1 << 30) * 132 * 4


def test_cpu_tensors_are_refused():
    c = ops.kv_cache_fp8(1, 2, "cpu")
    assert c[0].shape == (1, 2, 256, 128) and c[0].dtype == torch.float8_e4m3fn and c[2].shape == (1, 2, 4)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.NativeError, match="CUDA"):
        ops.paged_decode_attention_fp8(torch.zeros(1, 4, 128, dtype=torch.bfloat16), *c, i.view(1, 1), i, 0.1)


@pytest.mark.parametrize("batch", [0, 1, 7, 64, 512, 5000])
@pytest.mark.parametrize("hkv", [1, 8])
@pytest.mark.parametrize("ctx", [0, 1, 64, 65, 1000, 40960, 1 << 20])
def test_plans_cover_the_context(batch, hkv, ctx):
    for split, n in [ops.decode_split_plan_fp8(batch, hkv, ctx)]:
        assert split % 64 == 0 and 64 <= split <= 8192 and n >= 1 and split * n >= ctx and (n - 1) * split < max(1, ctx)
    step, sh, ns, ow, no = ops.grouped_decode_plan_fp8(batch, max(1, batch // 8), 2 * hkv, hkv, ctx, ctx)
    assert step == max(1, batch // 8)
    for split, n in ((sh, ns), (ow, no)):
        assert split % 64 == 0 and 64 <= split <= 8192 and n >= 1 and split * n >= ctx

@pytest.mark.parametrize("batch,total_q,max_q", [(1, 1, 1), (1, 20, 20), (4, 40, 30), (64, 64, 1), (1, 2048, 2048), (300, 300, 1)])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (16, 1), (8, 8)])
@pytest.mark.parametrize("max_k", [1, 511, 1025, 32768, 40961])
def test_prefill_plan_covers_the_keys(batch, total_q, max_q, hq, hkv, max_k):
    split, n = ops.prefill_split_plan_fp8(batch, total_q, max_q, max_k, hq, hkv)
    assert (split, n) == (0, 1) or (split % 128 == 0 and n > 1 and (n - 1) * split < max_k <= n * split)


def test_automatic_page_count_follows_the_cache_format(monkeypatch):
    """A pool sized to what memory holds is sized anew when the format changes (its pages take another number of
    bytes), after the old pool has been let go; a count that the user set stays."""
    from qwen3_naive_inference_b200.qwen3_naive import Qwen3Config, Qwen3ForCausalLM
    model = Qwen3ForCausalLM(Qwen3Config(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=128,
                                         intermediate_size=64, num_hidden_layers=2, vocab_size=32, max_position_embeddings=512))
    at = model.model.layers[1].self_attn
    budget, asked = 20 * 2 * 2 * 256 * 128 * 2, []

    def count():
        assert at.k_cache is None and at.v_scale is None and not model._has_cuda_graphs
        asked.append(model.kv_cache_dtype)
        return budget // model._block_bytes()

    monkeypatch.setattr(model, "_compute_num_blocks", count)

    def pool():
        model.allocate_global_kv_cache()
        t = [c for c in (at.k_cache, at.v_cache, at.k_scale, at.v_scale) if c is not None]
        assert all(c.shape[0] == model._num_blocks for c in t)
        return 2 * sum(c.numel() * c.element_size() for c in t)

    for dtype, pages in (("bf16", 20), ("fp8", 39), ("bf16", 20), ("fp8", 39)):
        model.kv_cache_dtype = dtype
        model._has_cuda_graphs = at.k_cache is not None
        assert pool() <= budget and model._num_blocks == pages
        kept = at.k_cache
        assert pool() <= budget and at.k_cache is kept  # nothing changed: the pool stays
    assert asked == ["bf16", "fp8", "bf16", "fp8"]
    model._num_blocks = 7  # the user's
    for dtype in ("bf16", "fp8", "bf16"):
        model.kv_cache_dtype = dtype
        pool()
        assert model._num_blocks == 7 and asked[4:] == []
