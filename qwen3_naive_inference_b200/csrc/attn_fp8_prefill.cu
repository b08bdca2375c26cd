// Attention over the 8-bit paged KV cache (kv_fp8.cuh): decode, grouped decode, prefill.
//
//   o = sum_j p_j vs_j V_j,   p = softmax_j(scale * ks_j * q . K_j)
//
// K_j, V_j the e4m3 codes of key j, ks_j, vs_j the scales of its block and head.
#include "attn_fp8.cuh"

namespace {

struct RowParams {
  const bf16* q;
  int64_t q_stride;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_width;
  const int32_t* seqlens;
  int seqlen_add;
  int batch, hq, hkv;  // batch: table rows
  float scale_log2;
  int n_groups;
  const int32_t* members;
  const int32_t* shared_len;
  const int32_t* kv_start;
  const int32_t* cu_q;
  const int32_t* cu_k;
  bf16* out;
  int64_t out_stride;
  int* err;
};

struct RowState {
  float q[4], o[4], m, l;
};

// Keys [a, b) of the pages of table row `tb` for one query row, one key at a time: a warp, four
// elements of the head a lane.
QB_DEVICE void row_keys(const RowParams& p, RowState& s, int64_t tb, int kvh, int a, int b, int lane) {
  for (int j = a; j < b; ++j) {
    const int w = j / KV8_PAGE;
    const int page = w < p.bt_width ? p.bt[tb * p.bt_stride + w] : -1;
    if (page < 0 || page >= p.num_blocks) {
      if (lane == 0) qb_set_err(p.err, QB_DEVERR_PAGE);
      continue;
    }
    const int64_t at = (int64_t)page * p.hkv + kvh;
    const int64_t row = (at * KV8_PAGE + j % KV8_PAGE) * KV8_D + lane * 4;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(p.k + row);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(p.v + row);
    const int sub = j % KV8_PAGE / KV8_BLOCK;
    const float2 k0 = e4m3x2_to_float2(kw & 0xffffu), k1 = e4m3x2_to_float2(kw >> 16);
    const float2 v0 = e4m3x2_to_float2(vw & 0xffffu), v1 = e4m3x2_to_float2(vw >> 16);
    float x = s.q[0] * k0.x + s.q[1] * k0.y + s.q[2] * k1.x + s.q[3] * k1.y;
    x = warp_sum(x) * p.ks[at * KV8_SUBS + sub] * p.scale_log2;
    const float m = fmaxf(s.m, x), alpha = exp2f(s.m - m), e = exp2f(x - m);
    const float ev = e * p.vs[at * KV8_SUBS + sub];
    s.m = m;
    s.l = s.l * alpha + e;
    s.o[0] = s.o[0] * alpha + ev * v0.x;
    s.o[1] = s.o[1] * alpha + ev * v0.y;
    s.o[2] = s.o[2] * alpha + ev * v1.x;
    s.o[3] = s.o[3] * alpha + ev * v1.y;
  }
}
QB_DEVICE void row_begin(const RowParams& p, RowState& s, int64_t row, int h, int lane) {
  const uint2 u = *reinterpret_cast<const uint2*>(p.q + row * p.q_stride + h * KV8_D + lane * 4);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
  s.q[0] = a.x; s.q[1] = a.y; s.q[2] = b.x; s.q[3] = b.y;
  s.o[0] = s.o[1] = s.o[2] = s.o[3] = 0.f;
  s.m = -INFINITY;
  s.l = 0.f;
}
QB_DEVICE void row_end(const RowParams& p, const RowState& s, int64_t row, int h, int lane) {
  const float inv = s.l > 0.f ? 1.f / s.l : (s.l == 0.f ? 0.f : s.l);
  uint2 u;
  u.x = pack_bf16x2(s.o[0] * inv, s.o[1] * inv);
  u.y = pack_bf16x2(s.o[2] * inv, s.o[3] * inv);
  *reinterpret_cast<uint2*>(p.out + row * p.out_stride + h * KV8_D + lane * 4) = u;
}

__global__ void __launch_bounds__(128)
prefill_rows_kernel(RowParams p, int64_t total) {
  qb_pdl_trigger();
  qb_pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int h = (int)(item % p.hq), kvh = h / (p.hq / p.hkv);
  const int64_t t = item / p.hq;
  if (t >= total) return;
  int b = 0;
  while (b < p.batch && p.cu_q[b + 1] <= t) ++b;
  if (b >= p.batch) return;
  const int lq = p.cu_q[b + 1] - p.cu_q[b], lk = p.cu_k[b + 1] - p.cu_k[b];
  if (lk < lq) {
    if (lane == 0) qb_set_err(p.err, QB_DEVERR_SHAPE);
    return;
  }
  RowState s;
  row_begin(p, s, t, h, lane);
  row_keys(p, s, b, kvh, 0, lk - lq + (int)(t - p.cu_q[b]) + 1, lane);
  row_end(p, s, t, h, lane);
}

}  // namespace

extern "C" int qb_attn_paged_prefill_fp8(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                                         const float* k_scale, const float* v_scale, int64_t num_blocks, int page_size,
                                         const int32_t* block_tables, int64_t bt_stride, int bt_width,
                                         const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                         const int32_t* tile_info, int n_tiles, int tiles_per_seq, int hq, int hkv,
                                         int D, float scale, void* out, int64_t o_stride, int64_t total_q, int* err,
                                         qb_stream_t stream) {
  if (D != KV8_D || page_size != KV8_PAGE) return QB_ERR_UNSUPPORTED;
  QB_CHECK_ARG(batch >= 0 && total_q >= 0 && total_q <= INT32_MAX && n_tiles >= 0 && tiles_per_seq >= 0);
  if (batch == 0 || total_q == 0) return QB_OK;
  const int st = kv8_check_cache(q, q_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_tables, bt_stride, bt_width,
                             hq, hkv, out);
  if (st != QB_OK) return st;
  QB_CHECK_ARG(cu_seqlens_q && cu_seqlens_k && o_stride >= (int64_t)hq * KV8_D && o_stride % 8 == 0);
  (void)tile_info;
  RowParams p{(const bf16*)q, q_stride, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, num_blocks,
              block_tables, bt_stride, bt_width, nullptr, 0, batch, hq, hkv, scale * KV8_LOG2E, 0, nullptr, nullptr, nullptr,
              cu_seqlens_q, cu_seqlens_k, (bf16*)out, o_stride, err};
  return qb_launch(prefill_rows_kernel, dim3((unsigned)((total_q * hq + 3) / 4)), dim3(128), 0, (cudaStream_t)stream, 1,
                   p, total_q);
}
