// QK-norm + RoPE of a projected token row with the append of its keys and values to the 8-bit paged
// cache (kv_fp8.cuh); the 8-bit form of the store in qk_norm_rope_fwd8_kernel.
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   (lo, hi) -> (lo c - hi s, hi c + lo s)      (fp32)
//
// Keys and values go from fp32 to e4m3 in one rounding (no bf16 in between); q is rounded to bf16.
// A block of 64 tokens and head has one scale: the smallest power of two under which everything
// appended since the block's first row stays within 448.  A power of two moves a code between scales
// without a rounding (but for codes that become subnormal, 2^-15 below the block's largest value),
// so a block may be filled a token at a time: where a later token raises the scale, the rows already
// there are rounded again under the new one.  A call that writes row 0 of a block begins it anew (a
// recycled page's old scale is dropped).
//
// Work split: a CTA per window of tokens and kv heads for K and V, further CTAs for q.  All tokens of the
// call that fall into one block are handled by the CTA whose window holds the first of them, so a block's
// scale has one writer; the CTA finds the others by scanning the slots (tokens whose left neighbour is in
// the same block never scan).  A slot given twice takes the later token.  Windows are 16 tokens in a
// decode step, where each token is in a block of its own (a warp each), 64 in long calls, where most are
// not, and as many heads share a scan as leave enough CTAs.
//
// Bound by HBM: 2 bytes read and 2 (q) or 1 (codes) written an element.  Measured on a B200 (16 query and 8 kv
// heads): one token 2.8 us; 512 tokens in 512 blocks 6.3 us (the rows and scales of a step are 8 MB: latency);
// 37 chunks, 10361 tokens, 45.4 us for 154 MB, 3.4 TB/s: a block's CTA loads, meets at a barrier for the scale and
// then stores, and two CTAs an SM overlap only in part.
#include <float.h>

#include "kv_fp8.cuh"

namespace {

constexpr int ST_THREADS = 512, ST_WARPS = ST_THREADS / 32, ST_HALVES = ST_THREADS / 16;
constexpr int ST_GROUP = ST_WARPS;             // tokens of a window in a short call, a warp each; blocks looked for at a time
constexpr int ST_LONG = 64;                    // tokens of a window in a long call ...
constexpr int ST_LONG_CALL = 768;              // ... of more tokens than a decode step has
constexpr int ST_ALONE_TRY = 8;                // more run heads than this in a window: look whether they are alone
constexpr int ST_ENOUGH = 512;                 // working K/V CTAs that keep the GPU busy
constexpr int ST_ROWS = KV8_BLOCK / ST_HALVES;  // rows of a block per half-warp
constexpr int ST_QH = 4;                       // q heads per half-warp item (one rotation-table row for all)

struct __align__(16) Row8 {  // eight bf16 of a head row
  uint32_t w[4];
};

struct StoreParams {
  const bf16* qkv;
  int64_t T, ld;
  int hq, hkv;
  const int64_t* positions;
  const float* cos_sin;
  int64_t max_pos;
  const bf16* qw;
  const bf16* kw;
  float eps;
  bf16* q_out;
  uint8_t* codes[2];  // K, V
  float* scales[2];
  const int32_t* slots;
  int64_t num_slots;
  int window, heads;  // tokens and kv heads of a K/V CTA
  int64_t n_kv_ctas;
  int* err;
};

QB_DEVICE Row8 ld_row(const bf16* p) { return *reinterpret_cast<const Row8*>(p); }
QB_DEVICE void unpack_row(const Row8& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(r.w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
QB_DEVICE float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
QB_DEVICE float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
QB_DEVICE int64_t checked_pos(const StoreParams& p, int64_t t, bool tell) {
  const int64_t pos = p.positions[t];
  if (pos >= 0 && pos < p.max_pos) return pos;
  if (tell) qb_set_err(p.err, QB_DEVERR_SHAPE);
  return 0;
}
// cos and sin of the eight rotation-table columns of lane l (columns j and j + 64 turn together: lo c - hi s
// in the lanes of the lower half, where s is given negated, hi c + lo s in those of the upper)
QB_DEVICE void ld_rotation(const StoreParams& p, int64_t pos, int l, float (&c)[8], float (&s)[8]) {
  const float* row = p.cos_sin + pos * KV8_D + (l & 7) * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 a = reinterpret_cast<const float4*>(row)[i];
    const float4 b = reinterpret_cast<const float4*>(row + KV8_D / 2)[i];
    c[4 * i] = a.x; c[4 * i + 1] = a.y; c[4 * i + 2] = a.z; c[4 * i + 3] = a.w;
    s[4 * i] = b.x; s[4 * i + 1] = b.y; s[4 * i + 2] = b.z; s[4 * i + 3] = b.w;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = l < 8 ? -s[i] : s[i];
}
// QK-norm and rotation of a head row spread over a half-warp (lane l: elements 8l..8l+7).  Every
// lane of the warp takes part in the shuffles.
QB_DEVICE void norm_rope(float (&v)[8], const float (&w)[8], const float (&c)[8], const float (&s)[8], float eps) {
  float2 sq = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) sq = fma2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(v[2 * i], v[2 * i + 1]), sq);
  const float rstd = qk_rstd(half_sum(sq.x + sq.y), eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = mul2(mul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(rstd, rstd)), make_float2(w[2 * i], w[2 * i + 1]));
    float2 partner;
    partner.x = __shfl_xor_sync(0xffffffffu, x.x, 8);
    partner.y = __shfl_xor_sync(0xffffffffu, x.y, 8);
    const float2 y = fma2(x, make_float2(c[2 * i], c[2 * i + 1]), mul2(partner, make_float2(s[2 * i], s[2 * i + 1])));
    v[2 * i] = y.x;
    v[2 * i + 1] = y.y;
  }
}
// Largest magnitude of a lane's values, as bits (they order as magnitudes do).  What is not finite is
// stored as NaN, whatever the scale, and does not count: `odd` says that there is such a value.
constexpr uint32_t FINITE = 0x7f7fffffu;
QB_DEVICE float finite_max(const float (&v)[8], bool& odd) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  odd = m > FINITE;
  if (odd) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
      m = max(m, a <= FINITE ? a : 0u);
    }
  }
  return __uint_as_float(m);
}
// Smallest power of two (at least 2^-126) under which `top` is within 448 = 1.75 * 2^8.
QB_DEVICE float scale_for(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}
QB_DEVICE void st_codes(uint8_t* dst, float (&v)[8], float inv, bool odd) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = mul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(inv, inv));
    v[2 * i] = y.x;
    v[2 * i + 1] = y.y;
  }
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((__float_as_uint(v[i]) & 0x7fffffffu) > FINITE) v[i] = __int_as_float(0x7fffffff);
  }
  uint2 u;
  u.x = float4_to_e4m3x4(v[0], v[1], v[2], v[3]);
  u.y = float4_to_e4m3x4(v[4], v[5], v[6], v[7]);
  *reinterpret_cast<uint2*>(dst) = u;
}
// Rounds the block's rows that this call does not write (`kept`) again under a scale larger by 1 / ratio.
// N threads take part, this one as number `i`.  Up to eight loads of a thread are on their way at once: in a decode
// step some block of the call nearly always needs it, and the step waits for that block's warp (one load after
// another: 22.8 us a call in a rollout of 512 sequences, 8.6 so).
template <int N, typename F>
QB_DEVICE void round_again(uint8_t* block, F kept, float ratio, int i) {
  constexpr int EACH = KV8_TILE / 16 / N, AHEAD = EACH < 8 ? EACH : 8;
  uint4* at = reinterpret_cast<uint4*>(block) + i;
#pragma unroll 1
  for (int c = 0; c < EACH; c += AHEAD) {
    uint4 u[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) u[k] = at[(c + k) * N];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        e4m3x4_to_float4(w[j], f);
        w[j] = float4_to_e4m3x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
      }
      if (kept((i + (c + k) * N) >> 3)) at[(c + k) * N] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
// The block's scale after values up to `top` joined it: the old one unless the block begins anew or
// `top` needs a larger one.
QB_DEVICE float joined_scale(float old, float top, bool anew) {
  const float need = scale_for(top);
  return anew ? need : fmaxf(old, need);
}

QB_DEVICE void store_q(const StoreParams& p, int64_t cta) {
  const int l = threadIdx.x & 15;
  const unsigned per_token = (p.hq + ST_QH - 1) / ST_QH, item = (unsigned)(cta * ST_HALVES) + (threadIdx.x >> 4);
  const bool live = item < (unsigned)p.T * per_token;
  const int64_t t = live ? item / per_token : 0;
  const int h0 = live ? (int)(item % per_token) * ST_QH : 0;
  Row8 raw[ST_QH];
#pragma unroll
  for (int k = 0; k < ST_QH; ++k)
    raw[k] = h0 + k < p.hq ? ld_row(p.qkv + t * p.ld + (h0 + k) * KV8_D + l * 8) : Row8{};
  float c[8], s[8], w[8];
  ld_rotation(p, checked_pos(p, t, live && l == 0), l, c, s);
  unpack_row(ld_row(p.qw + l * 8), w);
#pragma unroll
  for (int k = 0; k < ST_QH; ++k) {
    float v[8];
    unpack_row(raw[k], v);
    norm_rope(v, w, c, s, p.eps);
    if (live && h0 + k < p.hq) {
      Row8 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o.w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<Row8*>(p.q_out + (t * p.hq + h0 + k) * KV8_D + l * 8) = o;
    }
  }
}

// What a K/V CTA knows of up to ST_GROUP blocks whose first token may be in its window.
struct Found {
  int block[ST_GROUP];               // -1: none, or its first token is elsewhere
  int head[ST_GROUP];                // the run head that brought it
  int first[ST_GROUP];               // the call's first token in the block
  int row_src[ST_GROUP][KV8_BLOCK];  // the token that writes each row, -1: none
};

QB_DEVICE void note_match(Found& f, int i, int t, int slot) {
  atomicMin(&f.first[i], t);
  atomicMax(&f.row_src[i][slot & (KV8_BLOCK - 1)], t);
}
// Tokens of the call that fall into one of the n blocks.  A skipped slot (-1) matches no block.
QB_DEVICE void note_token(Found& f, int n, int t, int slot) {
  for (int i = 0; i < n; ++i)
    if (slot >> 6 == f.block[i]) note_match(f, i, t, slot);
}
QB_DEVICE void note_tokens(Found& f, int n, int t, const int4& s) {
  for (int i = 0; i < n; ++i) {  // one block, in a prompt chunk: four comparisons for four tokens
    const int blk = f.block[i];
    const bool a = s.x >> 6 == blk, b = s.y >> 6 == blk, c = s.z >> 6 == blk, d = s.w >> 6 == blk;
    if (a || b || c || d) {
      if (a) note_match(f, i, t, s.x);
      if (b) note_match(f, i, t + 1, s.y);
      if (c) note_match(f, i, t + 2, s.z);
      if (d) note_match(f, i, t + 3, s.w);
    }
  }
}

// A token that is alone in its block (a decode step): a warp, its first half K, its second half V.  The
// token's row, rotation and scale are on their way while the warp looks through the call's slots.  False
// where the block takes other tokens of the call, too: nothing is stored then.
QB_DEVICE bool store_alone(const StoreParams& p, int64_t t, int slot, int head, const float (&kw)[8], bool aligned) {
  const int lane = threadIdx.x & 31, l = lane & 15, which = lane >> 4, blk = slot >> 6, row = slot & (KV8_BLOCK - 1);
  const int64_t at = ((int64_t)(blk / KV8_SUBS) * p.hkv + head) * KV8_SUBS + blk % KV8_SUBS;
  float* scale = p.scales[which] + at;
  uint8_t* block = p.codes[which] + at * KV8_TILE;
  const Row8 raw = ld_row(p.qkv + t * p.ld + (p.hq + (which ? p.hkv : 0) + head) * KV8_D + l * 8);
  const float old = *scale;
  float v[8], y[8], c[8], s[8];
  ld_rotation(p, checked_pos(p, t, false), l, c, s);
  bool alone = true;
  const int quads = aligned ? (int)(p.T / 4) : 0;
#pragma unroll 4
  for (int i = lane; i < quads; i += 32) {
    const int4 o = reinterpret_cast<const int4*>(p.slots)[i];
    const int n = (o.x >> 6 == blk) + (o.y >> 6 == blk) + (o.z >> 6 == blk) + (o.w >> 6 == blk);
    alone = alone && n == (t >> 2 == i ? 1 : 0);
  }
  for (int i = 4 * quads + lane; i < (int)p.T; i += 32) alone = alone && (p.slots[i] >> 6 != blk || i == (int)t);
  if (!__all_sync(0xffffffffu, alone)) return false;
  unpack_row(raw, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = v[i];
  norm_rope(y, kw, c, s, p.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = which ? v[i] : y[i];
  const bool anew = row == 0;
  bool odd;
  const float now = joined_scale(old, half_max(finite_max(v, odd)), anew);
  st_codes(block + row * KV8_D + l * 8, v, 1.f / now, odd);
  if (l == 0) *scale = now;
  const unsigned raised = __ballot_sync(0xffffffffu, !anew && now > old);
#pragma unroll
  for (int side = 0; side < 2; ++side)
    if (raised >> (16 * side) & 1) {  // the whole warp, K's block, then V's
      const float ratio = __shfl_sync(0xffffffffu, old / now, 16 * side);
      round_again<32>(p.codes[side] + at * KV8_TILE, [row](int r) { return r != row; }, ratio, lane);
    }
  return true;
}

// A block that takes several tokens (a prompt chunk): 32 half-warps on 64 rows.
QB_DEVICE void store_many(const StoreParams& p, const Found& f, int i, int head, const float (&kw)[8], unsigned* top) {
  const int tid = threadIdx.x, lane = tid & 31, l = tid & 15, blk = f.block[i];
  __syncthreads();  // `top` of the block before has been read
  if (tid < 2) top[tid] = 0;
  __syncthreads();
  const int64_t at = ((int64_t)(blk / KV8_SUBS) * p.hkv + head) * KV8_SUBS + blk % KV8_SUBS;
  const int kcol = (p.hq + head) * KV8_D + l * 8, vcol = kcol + p.hkv * KV8_D;
  const float old_k = p.scales[0][at], old_v = p.scales[1][at];
  float k[ST_ROWS][8];
  Row8 v[ST_ROWS];
  float top_k = 0.f, top_v = 0.f;
  bool odd_k[ST_ROWS], odd_v[ST_ROWS];
#pragma unroll
  for (int r = 0; r < ST_ROWS; ++r) {
    const int64_t t = f.row_src[i][(tid >> 4) + r * ST_HALVES];
    const bool live = t >= 0;
    unpack_row(live ? ld_row(p.qkv + t * p.ld + kcol) : Row8{}, k[r]);
    v[r] = live ? ld_row(p.qkv + t * p.ld + vcol) : Row8{};
  }
#pragma unroll
  for (int r = 0; r < ST_ROWS; ++r) {
    const int64_t t = f.row_src[i][(tid >> 4) + r * ST_HALVES];
    float c[8], s[8];
    ld_rotation(p, t >= 0 ? checked_pos(p, t, false) : 0, l, c, s);
    norm_rope(k[r], kw, c, s, p.eps);
    float x[8];
    unpack_row(v[r], x);
    top_k = fmaxf(top_k, finite_max(k[r], odd_k[r]));  // a row not written is zero
    top_v = fmaxf(top_v, finite_max(x, odd_v[r]));
  }
  top_k = warp_max(top_k);
  top_v = warp_max(top_v);
  if (lane == 0) {  // magnitudes are not negative: their bits order as they do
    atomicMax(&top[0], __float_as_uint(top_k));
    atomicMax(&top[1], __float_as_uint(top_v));
  }
  __syncthreads();
  const bool anew = f.row_src[i][0] >= 0;
  const float now_k = joined_scale(old_k, __uint_as_float(top[0]), anew);
  const float now_v = joined_scale(old_v, __uint_as_float(top[1]), anew);
  uint8_t* kb = p.codes[0] + at * KV8_TILE;
  uint8_t* vb = p.codes[1] + at * KV8_TILE;
#pragma unroll
  for (int r = 0; r < ST_ROWS; ++r) {
    const int row = (tid >> 4) + r * ST_HALVES;
    if (f.row_src[i][row] < 0) continue;
    float x[8];
    unpack_row(v[r], x);
    st_codes(kb + row * KV8_D + l * 8, k[r], 1.f / now_k, odd_k[r]);
    st_codes(vb + row * KV8_D + l * 8, x, 1.f / now_v, odd_v[r]);
  }
  const auto kept = [&f, i](int r) { return f.row_src[i][r] < 0; };
  if (!anew && now_k > old_k) round_again<ST_THREADS>(kb, kept, old_k / now_k, tid);
  if (!anew && now_v > old_v) round_again<ST_THREADS>(vb, kept, old_v / now_v, tid);
  if (tid == 0) {
    p.scales[0][at] = now_k;
    p.scales[1][at] = now_v;
  }
}

__global__ void __launch_bounds__(ST_THREADS, 2)
kv_fp8_store_kernel(StoreParams p) {
  qb_pdl_trigger();
  qb_pdl_wait();
  __shared__ Found f;
  __shared__ int heads[ST_LONG], n_heads;  // run heads of the window: tokens whose left neighbour is in another block
  __shared__ unsigned top[2];
  if ((int64_t)blockIdx.x >= p.n_kv_ctas) {
    store_q(p, (int64_t)blockIdx.x - p.n_kv_ctas);
    return;
  }
  const unsigned kv = blockIdx.x;
  const int tid = threadIdx.x, head_groups = (p.hkv + p.heads - 1) / p.heads;
  const int head0 = (int)(kv % head_groups) * p.heads, head1 = min(p.hkv, head0 + p.heads);
  const int64_t t0 = (int64_t)(kv / head_groups) * p.window;
  const bool aligned = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0;
  float kw[8];
  unpack_row(ld_row(p.kw + (tid & 15) * 8), kw);
  if (tid == 0) n_heads = 0;
  __syncthreads();
  {
    // short calls: a warp per token of the window (one head); long ones: a thread per token
    const bool by_warp = p.window == ST_GROUP;  // (then one kv head)
    const int64_t t = t0 + (by_warp ? tid >> 5 : tid);
    if ((by_warp || tid < p.window) && t < p.T) {
      const int slot = p.slots[t], before = t > 0 ? p.slots[t - 1] : -1;
      const bool mine = !by_warp || (tid & 31) == 0;
      if (slot >= 0 && slot < p.num_slots) {
        if (before >> 6 != slot >> 6 && !(by_warp && store_alone(p, t, slot, head0, kw, aligned)) && mine)
          heads[atomicAdd(&n_heads, 1)] = (int)t;
      } else if (slot != -1 && head0 == 0 && mine) {
        qb_set_err(p.err, QB_DEVERR_SLOT);
      }
    }
  }
  __syncthreads();
  int n = n_heads;
  if (n > ST_ALONE_TRY) {
    // a long call whose tokens lie in blocks of their own (a large decode batch): a warp per token after all
    for (int i = tid >> 5; i < n; i += ST_WARPS) {
      const int t = heads[i];
      bool alone = true;
      for (int head = head0; alone && head < head1; ++head) alone = store_alone(p, t, p.slots[t], head, kw, aligned);
      if (alone && (tid & 31) == 0) heads[i] = -1;
    }
    __syncthreads();
    if (tid == 0) {
      n_heads = 0;
      for (int i = 0; i < n; ++i)
        if (heads[i] >= 0) heads[n_heads++] = heads[i];
    }
    __syncthreads();
    n = n_heads;
  }
  if (n == 0) return;
  for (int g0 = 0; g0 < n; g0 += ST_GROUP) {
    const int m = min(ST_GROUP, n - g0);
    __syncthreads();  // the group before is done
    if (tid < ST_GROUP) {
      f.head[tid] = tid < m ? heads[g0 + tid] : -1;
      f.block[tid] = tid < m ? p.slots[f.head[tid]] >> 6 : -1;
      f.first[tid] = INT32_MAX;
    }
    for (int i = tid; i < ST_GROUP * KV8_BLOCK; i += ST_THREADS) (&f.row_src[0][0])[i] = -1;
    __syncthreads();
    // every token of the call in one of those blocks
    const int quads = aligned ? (int)(p.T / 4) : 0;
#pragma unroll 4
    for (int t = tid; t < quads; t += ST_THREADS)
      note_tokens(f, m, 4 * t, reinterpret_cast<const int4*>(p.slots)[t]);
    for (int t = 4 * quads + tid; t < (int)p.T; t += ST_THREADS) note_token(f, m, t, p.slots[t]);
    __syncthreads();
    if (tid < ST_GROUP && f.block[tid] >= 0 && f.first[tid] != f.head[tid]) f.block[tid] = -1;  // another run head came first
    __syncthreads();
    for (int i = 0; i < m; ++i)
      if (f.block[i] >= 0)  // uniform across the CTA
        for (int head = head0; head < head1; ++head) store_many(p, f, i, head, kw, top);
  }
}

}  // namespace

extern "C" int qb_qk_norm_rope_store_fp8(const void* qkv, int64_t T, int64_t ld_in, int hq, int hkv, int D,
                                         const int64_t* positions, const float* cos_sin, int64_t max_pos,
                                         const void* q_norm_w, const void* k_norm_w, float eps, void* q_out,
                                         void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                         const int32_t* slot_mapping, int64_t num_blocks, int page_size, int* err,
                                         qb_stream_t stream) {
  QB_CHECK_ARG(T >= 0 && hq > 0 && hkv > 0 && num_blocks >= 0 && max_pos > 0);
  if (D != KV8_D || page_size != KV8_PAGE) return QB_ERR_UNSUPPORTED;
  if (T == 0) return QB_OK;
  QB_CHECK_ARG(qkv && positions && cos_sin && q_norm_w && k_norm_w && q_out && slot_mapping);
  QB_CHECK_ARG(k_cache && v_cache && k_scale && v_scale);
  QB_CHECK_ARG(ld_in >= (int64_t)(hq + 2 * hkv) * KV8_D && ld_in % 8 == 0);
  const auto al16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  QB_CHECK_ARG(al16(qkv) && al16(cos_sin) && al16(q_norm_w) && al16(k_norm_w) && al16(q_out) && al16(k_cache) &&
               al16(v_cache));
  QB_CHECK_ARG(num_blocks <= (int64_t)INT32_MAX / KV8_PAGE);  // slots are int32
  StoreParams p{(const bf16*)qkv, T, ld_in, hq, hkv, positions, cos_sin, max_pos, (const bf16*)q_norm_w,
                (const bf16*)k_norm_w, eps, (bf16*)q_out, {(uint8_t*)k_cache, (uint8_t*)v_cache},
                {k_scale, v_scale}, slot_mapping, num_blocks * KV8_PAGE, ST_GROUP, 1, 0, err};
  if (T > ST_LONG_CALL) {
    p.window = ST_LONG;
    while (p.heads < hkv && T / KV8_BLOCK * hkv / (2 * p.heads) >= ST_ENOUGH) p.heads *= 2;
  }
  const int64_t kv = (T + p.window - 1) / p.window * ((hkv + p.heads - 1) / p.heads);
  const int64_t q = (T * ((hq + ST_QH - 1) / ST_QH) + ST_HALVES - 1) / ST_HALVES;
  QB_CHECK_ARG(T <= INT32_MAX / hq && kv + q <= INT32_MAX);
  p.n_kv_ctas = kv;
  return qb_launch(kv_fp8_store_kernel, dim3((unsigned)(kv + q)), dim3(ST_THREADS), 0, (cudaStream_t)stream, 1, p);
}
