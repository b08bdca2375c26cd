// Causal attention of query chunks over the 8-bit paged KV cache (kv_fp8.cuh) on tcgen05 + TMEM.
//
//   o_i = sum_j p_ij vs_j V_j,   p_i = softmax_j(scale * ks_j * q_i . K_j),   j <= Lk - Lq + i
//
// K_j, V_j the e4m3 codes of key j, ks_j, vs_j the scales of its block of 64 tokens and head.  Bound by
// the tensor pipe (4 * 128 flops per query, head and key) and, as near, by the exponentials.
//
// A CTA takes up to 256 query rows of one sequence and kv head -- row R is query position R / group, head
// R % group, so the group's heads share every key -- as two tiles of 128 rows, A and B, and walks the
// keys a block of 64 at a time:
//   warps 0-3, 4-7  softmax of tile A, of tile B: a thread per row
//   warps 8-11      convert: codes come from global memory two blocks ahead, become halves (exactly) and go
//                   to shared memory in the swizzled layout of the MMA operands (rings of four blocks)
//   warps 12, 13    issue S_A, S_B = Q_x K^T (both operands in shared memory)
//   warps 14, 15    issue O_A, O_B += P_x V (P_x from TMEM, over the columns of its S_x); each of the four
//                   waits for its own inputs only, so no wait holds up another's MMAs
// S_x has two buffers in TMEM, so the scores of block j + 1 are ready when the softmax is done with block
// j: the softmax warps never wait for the tensor pipe.  TMEM: four S buffers of 64 columns, O_A, O_B of 128.
// Q enters as halves scaled by a power of two per row (its largest value in [2^9, 2^10): bf16 values stay
// exact down to 2^-23 of it); ks and the softmax scale meet the fp32 scores.  What meets V is the
// probability weighed by its block's scale, P = vs 2^(x - ref) = 2^(x + log2 vs - ref), rounded to halves:
// a row's ref is set 7 below the largest x + log2 vs and moved when one passes it by 15, so P stays below 2^15
// and loses nothing above 2^-31 of the largest share, however far apart the blocks' scales are.  The sum l
// has a reference of its own, moved by the same rule on x alone; a tile joins it as sum(P) 2^(ref - log2 vs - lref).
// A tile whose shares are all below 2^-100 of the reference (a block of zeros under the smallest scale, say) may
// still hold probability: it gives P = 0 and its sum is taken from 2^(x - lref).
// Keys behind a row's last one take a score of -inf; their V must not count either, so codes past the
// sequence are zeroed and, in tiles that some row sees in part, NaN codes of V are zeroed too and their
// keys noted: in a row that does attend such a key its NaN elements become NaN at the end (the codes are read once
// more), as the product makes them in tiles that every row sees.
// Few rows over many keys: the keys are split over CTAs, which write normalised partial outputs and the
// rows' log-sums for a second kernel to join.
//
// Measured on a B200 (16 query and 8 kv heads):
//   2048 queries over 32768 keys        562 to 572 us by box, 533 GFLOP: 940 TFLOP/s (a plain matrix product: 1662)
//   2048 over 8192                      150 us: 800 TFLOP/s
//   8 fresh prompts of 256 to 512       35.5 us; 11 short sequences 18.6 us: a CTA's start, first tile and end,
//                                       8 us of every call
// Of 2048 over 8192: tensor pipe and exponential unit are busy 46 and 47% of the time each, issue slots 47%.  No
// single one holds it up: without the exponentials it took 10% less, with an eighth of the MMAs 5%.  What a softmax
// warp does to a tile -- load, maximum, exponentials, store, each waiting for the one before -- is the period, about
// 2200 cycles, of which the exponential unit needs 1024 for its two warps.  Turns at that unit, eight converter warps,
// more registers for the softmax (setmaxnreg) and results written out through shared memory were all slower.
// Every wait is bounded (~2 s): on timeout QB_DEVERR_TIMEOUT is raised, all roles leave, TMEM is freed.
#include <float.h>

#include <algorithm>

#include "attn_fp8.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int PF_KEYS = KV8_BLOCK;                 // keys of a tile: one block, one ks, one vs
constexpr int PF_ROWS = 128;                       // rows of a query tile
constexpr int PF_THREADS = 16 * 32;
constexpr int PF_Q_HALF = PF_ROWS * 64 * 2, PF_Q_TILE = 2 * PF_Q_HALF;  // element halves 0-63, 64-127
constexpr int PF_KV_HALF = PF_KEYS * 64 * 2, PF_KV_TILE = 2 * PF_KV_HALF;
constexpr int PF_STAGES = 4;
constexpr int PF_Q = 0, PF_K = 2 * PF_Q_TILE, PF_V = PF_K + PF_STAGES * PF_KV_TILE;
constexpr int PF_META = PF_V + PF_STAGES * PF_KV_TILE;
constexpr int PF_SLOTS = 8, PF_SLOT = 4;           // tiles whose scales are held, words of one
constexpr int PF_BARS = 4 * PF_STAGES + 20;
// barriers; TMEM slot, abort flag; row factors; per slot the tile's scales and NaN keys; what the end needs
constexpr int PF_KEPT = PF_META + PF_BARS * 8 + 8 + 2 * PF_ROWS * 4 + PF_SLOTS * PF_SLOT * 4, PF_KEPT_BYTES = 64;
constexpr int PF_SMEM = PF_KEPT + PF_KEPT_BYTES + 1024 /*align*/;
constexpr uint32_t PF_COL_S = 0, PF_COL_O = 256;   // S: + 128 * query tile + 64 * buffer; O: + 128 * query tile
constexpr float PF_HEAD = 7.f, PF_SLACK = 15.f;    // ref = largest - 7; moves when one is above ref + 15
constexpr float PF_APART = -100.f;                 // log2 of a share of O below which P is taken as zero
constexpr int PF_WS_ROW = KV8_D + 4;

// kind::f16, D fp32, A and B f16, M = 128; S: N = 64, both K-major; O: N = 128, B (V) MN-major.
constexpr uint32_t PF_IDESC_S = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t PF_IDESC_O = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

struct PrefillP {
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
  int table_keys;        // that a row of the table can name
  const int32_t* cu_q;
  const int32_t* cu_k;
  int batch;
  const int32_t* tiles;  // nullable [n_tiles, 2]: (sequence, first row of a 64-row tile)
  int n_tiles;
  int tiles_per_seq;     // without tiles: of `unit` rows
  int hq, hkv, pos_per_cta, unit;  // unit = max(64, pos_per_cta): rows a grid tile stands for
  float scale_log2;
  int split_keys, n_splits;
  float* ws;
  bf16* out;
  int64_t o_stride;
  int64_t total_q;
  int* err;
};

QB_DEVICE uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
QB_DEVICE float max3(float a, float b, float c) {  // NaN only if all are
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
QB_DEVICE void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
QB_DEVICE void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk c (of 16) of row r of a tile of halves in the swizzled operand layout, its element halves
// `half` bytes apart
QB_DEVICE uint32_t operand_chunk(int r, int c, int half) {
  return (uint32_t)((c >> 3) * half + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// What a CTA works on.
struct PrefillWork {
  int b, q0, lq, shift, kvh;  // sequence, first query position, queries, Lk - Lq
  int64_t row0;               // row of the sequence's first query
  int rows, begin, end;       // query rows; keys [begin, end)
  int n[2];                   // key tiles of query tiles A and B
};
// What the end of a CTA needs of it, so that nobody holds it in registers until then.
struct PrefillKept {
  PrefillWork work;
  int nan;  // has a converter taken out a NaN value?
};
static_assert(sizeof(PrefillKept) <= PF_KEPT_BYTES && PF_KEPT % alignof(PrefillKept) == 0, "layout");

struct PrefillSmem {
  uint32_t base;
  uint8_t* ptr;
  QB_DEVICE uint32_t q(int x) const { return base + PF_Q + x * PF_Q_TILE; }
  QB_DEVICE uint32_t k(int j) const { return base + PF_K + j % PF_STAGES * PF_KV_TILE; }
  QB_DEVICE uint32_t v(int j) const { return base + PF_V + j % PF_STAGES * PF_KV_TILE; }
  // barriers; those of key tile j, and the phase of the ring that j is in
  QB_DEVICE uint32_t bar(int i) const { return base + PF_META + 8 * i; }
  QB_DEVICE uint32_t k_full(int j) const { return bar(j % PF_STAGES); }
  QB_DEVICE uint32_t k_empty(int j) const { return bar(PF_STAGES + j % PF_STAGES); }
  QB_DEVICE uint32_t v_full(int j) const { return bar(2 * PF_STAGES + j % PF_STAGES); }
  QB_DEVICE uint32_t v_empty(int j) const { return bar(3 * PF_STAGES + j % PF_STAGES); }
  QB_DEVICE uint32_t phase(int j) const { return (uint32_t)(j / PF_STAGES) & 1u; }
  // A waiter tells a barrier's phases apart by their parity, so it may be one phase late and no more.  S, P
  // and P V of tile j + 1 can be complete before those of j have been waited for, so each has a barrier per
  // buffer, whose next phase (tile j + 2) does not begin without the waiter.  Phase of tile j: j / 2.
  QB_DEVICE uint32_t s_full(int x, int j) const { return bar(4 * PF_STAGES + 2 * x + (j & 1)); }
  QB_DEVICE uint32_t p_ready(int x, int j) const { return bar(4 * PF_STAGES + 4 + 2 * x + (j & 1)); }
  QB_DEVICE uint32_t pv_done(int x, int j) const { return bar(4 * PF_STAGES + 8 + 2 * x + (j & 1)); }
  QB_DEVICE uint32_t buffer_phase(int j) const { return (uint32_t)(j >> 1) & 1u; }
  QB_DEVICE uint32_t o_last(int x) const { return bar(4 * PF_STAGES + 12 + x); }  // the last tile's P V
  QB_DEVICE uint32_t q_full(int x) const { return bar(4 * PF_STAGES + 14 + x); }
  QB_DEVICE uint32_t all_done(int i) const { return bar(4 * PF_STAGES + 16 + i); }
  QB_DEVICE uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(ptr + PF_META + 8 * PF_BARS); }
  QB_DEVICE volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(tmem_slot() + 1); }
  QB_DEVICE float* row_fac() const { return reinterpret_cast<float*>(tmem_slot() + 2); }
  // slot of key tile j: [0] ks (negative: no such page), [1] log2 vs; [2], [3] bits of NaN keys.
  // Eight slots: a slot is written for tile j + 8 when S of j + 4 is done, so the softmax is past j + 2.
  QB_DEVICE float* scales(int j) const { return row_fac() + 2 * PF_ROWS + j % PF_SLOTS * PF_SLOT; }
  QB_DEVICE uint32_t* nan_keys(int j) const { return reinterpret_cast<uint32_t*>(scales(j) + 2); }
  QB_DEVICE PrefillKept* kept() const { return reinterpret_cast<PrefillKept*>(ptr + PF_KEPT); }
};

// Sixteen codes as halves into chunks 2c and 2c + 1 of row r.
QB_DEVICE void put_codes(uint32_t tile, int r, int c, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) e4m3x4_to_half2x2(w[i], h[2 * i], h[2 * i + 1]);
  const uint32_t at = tile + operand_chunk(r, 2 * c, PF_KV_HALF);
  st_shared16(at, h[0], h[1], h[2], h[3]);
  st_shared16(at ^ 16u, h[4], h[5], h[6], h[7]);
}
// Bits 7 of the bytes of w that hold a NaN code.
QB_DEVICE uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// ------------------------------------------------------------------ converters
QB_DEVICE void prefill_convert(const PrefillP& p, const PrefillSmem& sm, const PrefillWork& w) {
  const int tid = threadIdx.x - 8 * 32, n = max(w.n[0], w.n[1]);
  // keys row0 + 16 i, i < 4; eight threads in a row store to eight different bank groups: even chunks of
  // one element half of two neighbouring keys
  const int chunk = (tid & 3) | ((tid >> 1) & 4), row0 = ((tid >> 4) << 1) | ((tid >> 2) & 1);
  const int first_masked = w.shift + w.q0 + 1;  // keys from here on are behind the first row's last one
  // A key tile on its way: its codes in registers (rows past the keys and tiles without a page: zero) and, in
  // thread 0, its scales.  Two tiles are, so that a tile's loads have the time of two to arrive; the page of
  // the one after them is looked up meanwhile.
  struct Coming {
    uint4 k[4], v[4];
    int64_t at;  // (page, head, block), -1: no page
    float ks, vs;
  };
  auto page_of = [&](int j) {
    const int col = (w.begin + j * PF_KEYS) / KV8_PAGE;
    return j < n && col < p.bt_width ? p.bt[(int64_t)w.b * p.bt_stride + col] : -1;
  };
  auto find = [&](Coming& c, int j, int page) {
    c.at = -1;
    if (page >= 0 && page < p.num_blocks)
      c.at = ((int64_t)page * p.hkv + w.kvh) * KV8_SUBS + (w.begin + j * PF_KEYS) % KV8_PAGE / KV8_BLOCK;
    else if (j < n && tid == 0)
      qb_set_err(p.err, QB_DEVERR_PAGE);
    c.ks = tid == 0 && c.at >= 0 ? p.ks[c.at] : -1.f;
    c.vs = tid == 0 && c.at >= 0 ? p.vs[c.at] : 0.f;
  };
  auto load = [&](const uint8_t* codes, uint4 (&r)[4], int64_t at, int j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = row0 + 16 * i;
      r[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0 && w.begin + j * PF_KEYS + key < w.end)
        r[i] = *reinterpret_cast<const uint4*>(codes + at * KV8_TILE + key * KV8_D + chunk * 16);
    }
  };
  int page = -1;  // of the tile after the two
  auto take = [&](Coming& c, int j) {
    const int later = page_of(j + 3);
    if (!mbar_wait(sm.k_empty(j), sm.phase(j) ^ 1, sm.abort_flag(), p.err)) return false;
    if (tid == 0) {
      float* sc = sm.scales(j);
      sc[0] = c.ks;
      sc[1] = log2f(c.vs);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) put_codes(sm.k(j), row0 + 16 * i, chunk, c.k[i]);
    fence_async_shared();
    mbar_arrive(sm.k_full(j));
    find(c, j + 2, page);
    load(p.k, c.k, c.at, j + 2);
    if (!mbar_wait(sm.v_empty(j), sm.phase(j) ^ 1, sm.abort_flag(), p.err)) return false;
    if (w.begin + (j + 1) * PF_KEYS > first_masked) {
      // some row sees this tile in part: no NaN may reach the product of a masked key
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bad[4] = {nan_bytes(c.v[i].x), nan_bytes(c.v[i].y), nan_bytes(c.v[i].z), nan_bytes(c.v[i].w)};
        if (bad[0] | bad[1] | bad[2] | bad[3]) {
          c.v[i].x &= ~((bad[0] >> 7) * 0xffu);
          c.v[i].y &= ~((bad[1] >> 7) * 0xffu);
          c.v[i].z &= ~((bad[2] >> 7) * 0xffu);
          c.v[i].w &= ~((bad[3] >> 7) * 0xffu);
          const int key = row0 + 16 * i;
          atomicOr(&sm.nan_keys(j)[key >> 5], 1u << (key & 31));
          sm.kept()->nan = 1;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) put_codes(sm.v(j), row0 + 16 * i, chunk, c.v[i]);
    fence_async_shared();
    mbar_arrive(sm.v_full(j));
    load(p.v, c.v, c.at, j + 2);
    page = later;
    return true;
  };
  Coming a, b;
  const int page0 = page_of(0), page1 = page_of(1);
  page = page_of(2);
  find(a, 0, page0);
  load(p.k, a.k, a.at, 0);
  find(b, 1, page1);
  load(p.v, a.v, a.at, 0);
  load(p.k, b.k, b.at, 1);
  load(p.v, b.v, b.at, 1);
  for (int j = 0; j < n; j += 2) {
    if (!take(a, j)) return;
    if (j + 1 < n && !take(b, j + 1)) return;
  }
}

// ------------------------------------------------------------------ MMA issuers
// A warp for S and a warp for O of query tile x.  The whole warp walks the loop and one elected lane
// issues, so that what an MMA takes is computed once for the warp, in uniform registers: a single thread
// in the loop needs longer to issue the MMAs than the tensor pipe to execute them.
QB_DEVICE void prefill_issue(const PrefillP& p, const PrefillSmem& sm, const PrefillWork& w, uint32_t tmem, int x,
                             bool scores) {
  volatile int* ab = sm.abort_flag();
  const int n = max(w.n[0], w.n[1]), mine = w.n[x];
  uint32_t pred;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(pred));
  const bool one = pred != 0;
  auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, p.err)) != 0; };
  const uint32_t s_at = tmem + PF_COL_S + x * 128, o_at = tmem + PF_COL_O + x * 128;
  bool ok = true;
  if (scores) {
    const uint64_t q = sw128_kmajor_desc(sm.q(x)), k0 = sw128_kmajor_desc(sm.k(0));
    ok = mine == 0 || wait(sm.q_full(x), 0);
    for (int j = 0; ok && j < n; ++j) {
      if (!(ok = wait(sm.k_full(j), sm.phase(j)))) break;
      if (j >= mine) {  // past this query tile's last key: the stage is free as far as it goes
        if (one) mbar_arrive(sm.k_empty(j));
        continue;
      }
      // the buffer held P of j - 2
      if (j >= 2 && !(ok = wait(sm.pv_done(x, j), sm.buffer_phase(j - 2)))) break;
      tc_fence_after();
      if (one) {
        const uint64_t k = k0 + (uint64_t)(j % PF_STAGES * (PF_KV_TILE >> 4));
#pragma unroll
        for (int i = 0; i < 8; ++i)  // 128 elements in steps of 16
          umma_bf16(s_at + (j & 1) * 64, q + (((i >> 2) * PF_Q_HALF + (i & 3) * 32) >> 4),
                    k + (((i >> 2) * PF_KV_HALF + (i & 3) * 32) >> 4), PF_IDESC_S, i > 0);
        umma_commit(sm.s_full(x, j));
        umma_commit(sm.k_empty(j));
      }
    }
  } else {
    const uint64_t v0 = sw128_mn_desc(sm.v(0), PF_KV_HALF);
    for (int j = 0; ok && j < n; ++j) {
      if (!(ok = wait(sm.v_full(j), sm.phase(j)))) break;
      if (j >= mine) {
        if (one) mbar_arrive(sm.v_empty(j));
        continue;
      }
      if (!(ok = wait(sm.p_ready(x, j), sm.buffer_phase(j)))) break;
      tc_fence_after();
      if (one) {
        const uint64_t v = v0 + (uint64_t)(j % PF_STAGES * (PF_KV_TILE >> 4));
#pragma unroll
        for (int i = 0; i < 4; ++i)  // 64 keys in steps of 16: P columns 8 i, V rows 16 i
          umma_bf16_ts(o_at, s_at + (j & 1) * 64 + 8 * i, v + ((i * 16 * 128) >> 4), PF_IDESC_O, (j > 0 || i > 0) ? 1u : 0u);
        umma_commit(sm.pv_done(x, j));
        if (j + 1 == mine) umma_commit(sm.o_last(x));
        umma_commit(sm.v_empty(j));
      }
    }
  }
  // no MMA may still be reading shared memory or writing TMEM when the CTA leaves
  if (one) {
    const uint32_t done = sm.all_done(x + (scores ? 0 : 2));
    umma_commit(done);
    mbar_drain(done, 0);
  }
}

// ------------------------------------------------------------------ softmax
// Query tile x into shared memory as halves: a half-warp per row, 16 rows each.
QB_DEVICE void prefill_load_q(const PrefillP& p, const PrefillSmem& sm, const PrefillWork& w, int x) {
  const int tid = threadIdx.x & 127, l = tid & 15, group = p.hq / p.hkv;
  uint4 rows[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int R = x * PF_ROWS + (tid >> 4) + 8 * i;
    rows[i] = make_uint4(0, 0, 0, 0);
    if (R < w.rows)
      rows[i] = *reinterpret_cast<const uint4*>(p.q + (w.row0 + w.q0 + R / group) * p.q_stride +
                                                (w.kvh * group + R % group) * KV8_D + l * 8);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = (tid >> 4) + 8 * i, R = x * PF_ROWS + r;
    const uint4 u = rows[i];
    const uint32_t raw[4] = {u.x, u.y, u.z, u.w};
    float f[8], top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 g = unpack_bf16x2(raw[k]);
      f[2 * k] = g.x;
      f[2 * k + 1] = g.y;
      top = fmaxf(top, fmaxf(fabsf(g.x), fabsf(g.y)));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = max((int)(__float_as_uint(top) >> 23), 10);
    float mul = __uint_as_float((uint32_t)(263 - e) << 23);
    if (p.scale_log2 < 0.f) mul = -mul;  // the scores' factor is then positive
    if (l == 0) sm.row_fac()[R] = __uint_as_float((uint32_t)(e - 9) << 23) * fabsf(p.scale_log2);
    st_shared16(sm.q(x) + operand_chunk(r, l, PF_Q_HALF), pack_half2(f[0] * mul, f[1] * mul), pack_half2(f[2] * mul, f[3] * mul),
                pack_half2(f[4] * mul, f[5] * mul), pack_half2(f[6] * mul, f[7] * mul));
  }
  fence_async_shared();
}

QB_DEVICE void prefill_softmax(const PrefillP& p, const PrefillSmem& sm, const PrefillWork& w, uint32_t tmem, int x,
                               int split) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = (warp & 3) * 32 + lane, R = x * PF_ROWS + r;
  const int group = p.hq / p.hkv, n = w.n[x];
  if (n == 0) return;
  prefill_load_q(p, sm, w, x);
  mbar_arrive(sm.q_full(x));
  // the factors of this warp's rows come from other warps: wait for all 128 threads
  volatile int* ab = sm.abort_flag();
  bool ok = __all_sync(0xffffffffu, mbar_wait(sm.q_full(x), 0, ab, p.err));
  const float fac = ok ? sm.row_fac()[R] : 0.f;
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t o_at = lanes + PF_COL_O + x * 128;
  const bool live = R < w.rows;
  const int pos = w.q0 + R / group;
  // the row's last key here (rows behind the work's last do not hold the warp to the masked path)
  const int last = live ? min(w.shift + pos, w.end - 1) : w.end - 1;
  if (ok && __all_sync(0xffffffffu, !live)) {
    // nothing to weigh: what stands in these lanes of TMEM meets their own rows of O only
    for (int j = 0; ok && j < n; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(sm.s_full(x, j), sm.buffer_phase(j), ab, p.err)) != 0;
      if (ok) mbar_arrive(sm.p_ready(x, j));
    }
    return;
  }
  // O counts in units of 2^ref, l in units of 2^lref
  float ref = -INFINITY, lref = -INFINITY, l = 0.f;
  for (int j = 0; ok && j < n; ++j) {
    // tcgen05 loads and stores are warp-collective: every decision that leads to them is warp-uniform
    if (!__all_sync(0xffffffffu, mbar_wait(sm.s_full(x, j), sm.buffer_phase(j), ab, p.err))) {
      ok = false;
      break;
    }
    tc_fence_after();
    const uint32_t s_at = lanes + PF_COL_S + x * 128 + (j & 1) * 64;
    uint32_t v[64];
    tmem_ld32_nowait(s_at, v);
    tmem_ld32_nowait(s_at + 32, v + 32);
    const float* sc = sm.scales(j);
    const float ks = sc[0], lvs = sc[1];
    const int seen = ks < 0.f ? 0 : last - (w.begin + j * PF_KEYS) + 1;  // keys of the tile that the row sees
    const float f = fmaxf(fac * ks, FLT_MIN);  // not zero: -inf (a key not seen) has to stay -inf
    const bool whole = __all_sync(0xffffffffu, seen >= PF_KEYS);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(v[i]));  // no use of a score moves above the wait
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 64; ++i)
        if (i >= seen) v[i] = __float_as_uint(-INFINITY);
    }
    float top[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) top[c] = max3(__uint_as_float(v[c]), __uint_as_float(v[c + 4]), __uint_as_float(v[c + 8]));
#pragma unroll
    for (int i = 12; i < 60; i += 8)
#pragma unroll
      for (int c = 0; c < 4; ++c) top[c] = max3(top[c], __uint_as_float(v[i + c]), __uint_as_float(v[i + 4 + c]));
#pragma unroll
    for (int c = 0; c < 4; ++c) top[c] = fmaxf(top[c], __uint_as_float(v[60 + c]));
    const float mt = f * fmaxf(max3(top[0], top[1], top[2]), top[3]), mw = mt + lvs;  // largest score, plain and weighed
    const bool need = mw > ref + PF_SLACK;
    if (__any_sync(0xffffffffu, need)) {
      float a = 1.f;
      if (need) {
        const float to = mw - PF_HEAD;
        a = ref == -INFINITY ? 0.f : fast_exp2(ref - to);
        ref = to;
      }
      if (j > 0) {  // O holds the tiles before: wait for the last of them, weigh them anew
        if (!__all_sync(0xffffffffu, mbar_wait(sm.pv_done(x, j - 1), sm.buffer_phase(j - 1), ab, p.err))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 128; c += 16) {
          uint32_t o[16];
          tmem_ld16(o_at + c, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
          tmem_st16(o_at + c, o);
        }
      }
    }
    if (mt > lref + PF_SLACK) {
      const float to = mt - PF_HEAD;
      l *= lref == -INFINITY ? 0.f : fast_exp2(lref - to);
      lref = to;
    }
    // does the row see keys here whose shares of O are all next to nothing?  (ref is -inf while every vs was zero)
    const bool apart = mt > -INFINITY && !(mw - ref >= PF_APART);
    const float shift = apart ? -lref : lvs - (ref == -INFINITY ? 0.f : ref);
    // takes a tile's sum to units of 2^lref; at most 2^115 where the tile is not `apart`
    const float to_l = apart ? 1.f : mt == -INFINITY ? 0.f : fast_exp2(ref - lvs - lref);
    const float2 ff = make_float2(f, f), ss = make_float2(shift, shift);
    float2 sum[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] = make_float2(0.f, 0.f);
    uint32_t pk[32];
    // Two loops, so that a score is not needed again once it is a probability: its register is free for the
    // ones that follow.
    if (!__any_sync(0xffffffffu, apart)) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float2 y = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ff, ss);
        y.x = fast_exp2(y.x);
        y.y = fast_exp2(y.y);
        sum[i & 3] = add2(sum[i & 3], y);
        pk[i] = pack_half2(y.x, y.y);
      }
    } else {  // some rows' probabilities go to the sum only
      const float keep = apart ? 0.f : 1.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float2 y = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ff, ss);
        y.x = fast_exp2(y.x);
        y.y = fast_exp2(y.y);
        sum[i & 3] = add2(sum[i & 3], y);
        pk[i] = pack_half2(y.x * keep, y.y * keep);
      }
    }
    tmem_st32(s_at, pk);
    const float2 s2 = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
    l = fmaf(s2.x + s2.y, to_l, l);
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(sm.p_ready(x, j));
  }
  if (!ok || !__all_sync(0xffffffffu, mbar_wait(sm.o_last(x), 0, ab, p.err))) return;
  tc_fence_after();
  // 2^(ref - lref) / l in two factors: value scales reach both ends of the exponent range
  const float units = ref == -INFINITY ? 0.f : ref - lref, half = rintf(0.5f * units), back = exp2f(half);
  const float inv = l == 0.f ? 0.f : exp2f(units - half) / l;
  const int64_t row = w.row0 + pos;
  const int head = w.kvh * group + R % group;
  bf16* out = p.out + row * p.o_stride + head * KV8_D;
  float* ws = p.ws + (p.n_splits > 1 ? ((row * p.hq + head) * p.n_splits + split) * PF_WS_ROW : 0);
#pragma unroll 1
  for (int c = 0; c < 128; c += 32) {
    uint32_t o[32];
    tmem_ld32(o_at + c, o);
    if (!live) continue;
    if (p.n_splits > 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<float4*>(ws + c)[i] =
            make_float4(__uint_as_float(o[4 * i]) * inv * back, __uint_as_float(o[4 * i + 1]) * inv * back,
                        __uint_as_float(o[4 * i + 2]) * inv * back, __uint_as_float(o[4 * i + 3]) * inv * back);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 u;
        u.x = pack_bf16x2(__uint_as_float(o[8 * i + 0]) * inv * back, __uint_as_float(o[8 * i + 1]) * inv * back);
        u.y = pack_bf16x2(__uint_as_float(o[8 * i + 2]) * inv * back, __uint_as_float(o[8 * i + 3]) * inv * back);
        u.z = pack_bf16x2(__uint_as_float(o[8 * i + 4]) * inv * back, __uint_as_float(o[8 * i + 5]) * inv * back);
        u.w = pack_bf16x2(__uint_as_float(o[8 * i + 6]) * inv * back, __uint_as_float(o[8 * i + 7]) * inv * back);
        reinterpret_cast<uint4*>(out + c)[i] = u;
      }
    }
  }
  if (live && p.n_splits > 1) ws[KV8_D] = l == 0.f ? -INFINITY : lref + log2f(l);
}

// NaN values that the converters took out of the tiles some row sees in part, into the elements of the rows that do
// attend them, after the rows have been written.  A thread per row and half of its elements.
QB_DEVICE void prefill_put_nan(const PrefillP& p, const PrefillSmem& sm, int split) {
  const PrefillWork w = sm.kept()->work;
  const int group = p.hq / p.hkv, R = threadIdx.x & 255, e0 = (threadIdx.x >> 8) * 64, n = w.n[R / PF_ROWS];
  if (R >= w.rows) return;
  const int64_t row = w.row0 + w.q0 + R / group;
  const int head = w.kvh * group + R % group, last = min(w.shift + w.q0 + R / group, w.end - 1);
  for (int j = max(0, w.shift + w.q0 + 1 - w.begin) / PF_KEYS; j < n; ++j)
    for (int k = 0; k < 2; ++k) {
      const int m = last - (w.begin + j * PF_KEYS + 32 * k) + 1;  // keys of the word that the row sees
      const uint32_t seen = m >= 32 ? 0xffffffffu : (m <= 0 ? 0u : (1u << m) - 1u);
      for (uint32_t keys = sm.nan_keys(j)[k] & seen; keys != 0; keys &= keys - 1) {
        const int key = w.begin + j * PF_KEYS + 32 * k + __ffs(keys) - 1;
        const int page = p.bt[(int64_t)w.b * p.bt_stride + key / KV8_PAGE];  // in the pool, or there would be no NaN
        const uint8_t* codes = p.v + (((int64_t)page * p.hkv + w.kvh) * KV8_PAGE + key % KV8_PAGE) * KV8_D;
        for (int e = e0; e < e0 + 64; ++e) {
          if ((codes[e] & 0x7f) != 0x7f) continue;
          if (p.n_splits > 1) p.ws[((row * p.hq + head) * p.n_splits + split) * PF_WS_ROW + e] = __int_as_float(0x7fffffff);
          else p.out[row * p.o_stride + head * KV8_D + e] = f2bf(__int_as_float(0x7fffffff));
        }
      }
    }
}

__global__ void __launch_bounds__(PF_THREADS, 1)
prefill_fp8_kernel(PrefillP p) {
  qb_pdl_wait();  // metadata and operands may come from the kernel before; also before any exit
  extern __shared__ uint8_t smem_raw[];
  PrefillWork w;
  const int group = p.hq / p.hkv, subs = p.unit / p.pos_per_cta;
  // the last tiles of the sequences, which see the most keys, begin first
  const int rank = gridDim.x - 1 - blockIdx.x, tile = rank / subs, sub = rank % subs, split = blockIdx.z;
  w.kvh = blockIdx.y;
  w.b = p.tiles ? p.tiles[2 * tile] : tile % p.batch;
  const int start = p.tiles ? p.tiles[2 * tile + 1] : tile / p.batch * p.unit;
  if (w.b < 0 || w.b >= p.batch || start < 0 || start % p.unit != 0) {
    // a 64-row tile whose rows belong to the CTA of an earlier one
    if ((w.b < 0 || w.b >= p.batch || start < 0) && threadIdx.x == 0) qb_set_err(p.err, QB_DEVERR_SHAPE);
    return;
  }
  w.row0 = p.cu_q[w.b];
  w.lq = p.cu_q[w.b + 1] - (int)w.row0;
  const int lk = p.cu_k[w.b + 1] - p.cu_k[w.b];
  w.q0 = start + sub * p.pos_per_cta;
  if (w.q0 >= w.lq) return;
  if (!p.tiles && w.q0 == 0 && w.lq / p.unit > p.tiles_per_seq - (w.lq % p.unit != 0) && threadIdx.x == 0)
    qb_set_err(p.err, QB_DEVERR_SHAPE);  // queries past the last tile
  if (lk < w.lq || w.row0 < 0 || w.row0 + w.lq > p.total_q) {
    if (threadIdx.x == 0) qb_set_err(p.err, QB_DEVERR_SHAPE);
    return;
  }
  w.shift = lk - w.lq;
  const int positions = min(p.pos_per_cta, w.lq - w.q0);
  w.rows = positions * group;
  w.begin = split * p.split_keys;
  w.end = min(w.shift + w.q0 + positions, p.n_splits > 1 ? w.begin + p.split_keys : INT32_MAX);
  if (p.n_splits > 1 && split == p.n_splits - 1 && w.end < w.shift + w.q0 + positions && threadIdx.x == 0)
    qb_set_err(p.err, QB_DEVERR_SHAPE);  // keys past the last split
  if (w.end > p.table_keys) {  // such keys are left out
    if (threadIdx.x == 0) qb_set_err(p.err, QB_DEVERR_PAGE);
    w.end = p.table_keys;
  }
  if (w.begin >= w.end) return;  // uniform across the CTA, before any barrier or TMEM exists
  const int rows_a = min(w.rows, PF_ROWS);
  const int end_a = min(w.end, w.shift + w.q0 + (rows_a - 1) / group + 1);  // tile A's last row's keys
  // tile A may see none of a late split's keys; a tile is kept all the same: its rows' sums are zero
  w.n[0] = (max(end_a - w.begin, 1) + PF_KEYS - 1) / PF_KEYS;
  w.n[1] = w.rows > PF_ROWS ? (w.end - w.begin + PF_KEYS - 1) / PF_KEYS : 0;

  PrefillSmem sm;
  const uint32_t raw = smem_u32(smem_raw);
  sm.base = (raw + 1023) & ~1023u;
  sm.ptr = smem_raw + (sm.base - raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < PF_STAGES; ++i) {
      mbar_init(sm.k_full(i), 128);
      mbar_init(sm.k_empty(i), 2);
      mbar_init(sm.v_full(i), 128);
      mbar_init(sm.v_empty(i), 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sm.q_full(i), 128);
      mbar_init(sm.o_last(i), 1);
      for (int k = 0; k < 2; ++k) {
        mbar_init(sm.s_full(i, k), 1);
        mbar_init(sm.p_ready(i, k), 128);
        mbar_init(sm.pv_done(i, k), 1);
        mbar_init(sm.all_done(2 * i + k), 1);
      }
    }
    *sm.abort_flag() = 0;
    // tiles that some row sees in part are the last five at most: their slots' NaN keys are written once
    for (int j = 0; j < PF_SLOTS; ++j) sm.nan_keys(j)[0] = sm.nan_keys(j)[1] = 0;
    sm.kept()->work = w;
    sm.kept()->nan = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(sm.tmem_slot())),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sm.tmem_slot();
  qb_pdl_trigger();  // after the TMEM allocation: the next kernel cannot take it from this CTA
  if (warp < 8) {
    prefill_softmax(p, sm, w, tmem, warp >> 2, split);
  } else if (warp < 12) {
    prefill_convert(p, sm, w);
  } else {
    prefill_issue(p, sm, w, tmem, warp & 1, warp < 14);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (__builtin_expect(sm.kept()->nan, 0)) prefill_put_nan(p, sm, split);
}

// Joins the key splits of a (row, head): a warp each, weights 2^(lse - largest lse), over the splits that
// hold keys of the row.  Rows of no tile have no partial outputs and are left as they are; the tiles of a call
// that is split are few (fewer than the GPU has SMs, in what prefill_split_plan_fp8 splits), so a warp looks
// through them.
__global__ void __launch_bounds__(128)
prefill_fp8_join_kernel(PrefillP p) {
  qb_pdl_trigger();
  qb_pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, head = (int)(item % p.hq);
  const int64_t row = item / p.hq;
  if (row >= p.total_q) return;
  int lo = 0, hi = p.batch;  // the sequence whose rows hold `row`: the last with cu_q <= row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.cu_q[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int lq = p.cu_q[lo + 1] - p.cu_q[lo], lk = p.cu_k[lo + 1] - p.cu_k[lo], i = (int)row - p.cu_q[lo];
  if (p.cu_q[lo] < 0 || i < 0 || i >= lq || lk < lq || p.cu_q[lo + 1] > p.total_q || p.table_keys == 0) return;
  bool tiled = i < (int64_t)p.tiles_per_seq * p.unit;
  if (p.tiles) {
    const int start = i & ~(p.unit - 1);  // of the grid tile that the row belongs to (unit is 64, 128 or 256)
    tiled = false;
    for (int k = lane; k < p.n_tiles; k += 32) tiled |= p.tiles[2 * k] == lo && p.tiles[2 * k + 1] == start;
    tiled = __any_sync(0xffffffffu, tiled);
  }
  if (!tiled) return;
  const int n = min(p.n_splits, min(lk - lq + i, p.table_keys - 1) / p.split_keys + 1);
  const float* ws = p.ws + (row * p.hq + head) * p.n_splits * PF_WS_ROW;
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, ws[(int64_t)s * PF_WS_ROW + KV8_D]);
  m = warp_max(m);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float* at = ws + (int64_t)s * PF_WS_ROW;
    const float lse = at[KV8_D], f = lse == -INFINITY ? 0.f : exp2f(lse - m);
    const float4 x = *reinterpret_cast<const float4*>(at + lane * 4);
    sum += f;
    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint2 u;
  u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + row * p.o_stride + head * KV8_D + lane * 4) = u;
}

}  // namespace

extern "C" size_t qb_attn_paged_prefill_fp8_workspace_bytes(int64_t total_q, int hq, int n_splits) {
  return n_splits <= 1 ? 0 : (size_t)total_q * hq * n_splits * PF_WS_ROW * 4;
}

extern "C" int qb_attn_paged_prefill_fp8(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                                         const float* k_scale, const float* v_scale, int64_t num_blocks, int page_size,
                                         const int32_t* block_tables, int64_t bt_stride, int bt_width,
                                         const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                         const int32_t* tile_info, int n_tiles, int tiles_per_seq, int hq, int hkv,
                                         int D, float scale, int split_keys, int n_splits, float* workspace, void* out,
                                         int64_t o_stride, int64_t total_q, int* err, qb_stream_t stream) {
  if (D != KV8_D || page_size != KV8_PAGE) return QB_ERR_UNSUPPORTED;
  QB_CHECK_ARG(batch >= 0 && total_q >= 0 && total_q <= INT32_MAX && n_tiles >= 0 && tiles_per_seq >= 0);
  QB_CHECK_ARG(n_splits >= 1 && n_splits <= 65535 && (n_splits == 1 || (split_keys > 0 && split_keys % (2 * PF_KEYS) == 0 &&
               (int64_t)split_keys * n_splits <= INT32_MAX / 2)));
  if (batch == 0 || total_q == 0) return QB_OK;
  const int ok = kv8_check_cache(q, q_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_tables, bt_stride,
                                 bt_width, hq, hkv, out);
  if (ok != QB_OK) return ok;
  QB_CHECK_ARG(cu_seqlens_q && cu_seqlens_k && o_stride >= (int64_t)hq * KV8_D && o_stride % 8 == 0 && hkv <= 65535);
  QB_CHECK_ARG(n_splits == 1 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0));
  PrefillP p{};
  p.q = (const bf16*)q; p.q_stride = q_stride; p.k = (const uint8_t*)k_cache; p.v = (const uint8_t*)v_cache;
  p.ks = k_scale; p.vs = v_scale; p.num_blocks = num_blocks; p.bt = block_tables; p.bt_stride = bt_stride;
  p.bt_width = bt_width; p.table_keys = (int)std::min<int64_t>((int64_t)bt_width * KV8_PAGE, INT32_MAX);
  p.cu_q = cu_seqlens_q; p.cu_k = cu_seqlens_k; p.batch = batch; p.tiles = tile_info; p.n_tiles = n_tiles;
  p.hq = hq; p.hkv = hkv;
  p.pos_per_cta = 16;
  while (p.pos_per_cta * 2 * (hq / hkv) <= 2 * PF_ROWS) p.pos_per_cta *= 2;
  p.unit = p.pos_per_cta > 64 ? p.pos_per_cta : 64;
  p.tiles_per_seq = (int)(((int64_t)tiles_per_seq * 64 + p.unit - 1) / p.unit);
  p.scale_log2 = scale * KV8_LOG2E;
  p.split_keys = n_splits > 1 ? split_keys : 0; p.n_splits = n_splits; p.ws = workspace; p.out = (bf16*)out;
  p.o_stride = o_stride; p.total_q = total_q; p.err = err;
  const int64_t grid = (tile_info ? (int64_t)n_tiles : (int64_t)batch * p.tiles_per_seq) * (p.unit / p.pos_per_cta);
  QB_CHECK_ARG(grid <= INT32_MAX);
  if (grid == 0) return QB_OK;
  static std::atomic<uint64_t> allowed{0};
  const int may = kv8_allow_smem(reinterpret_cast<const void*>(prefill_fp8_kernel), PF_SMEM, allowed);
  if (may != QB_OK) return may;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rc = qb_launch_ex(prefill_fp8_kernel, dim3((unsigned)grid, (unsigned)hkv, (unsigned)n_splits), dim3(PF_THREADS),
                              PF_SMEM, st, 1, true, p);
  if (rc != QB_OK || n_splits == 1) return rc;
  const int64_t items = total_q * hq;
  if ((items + 3) / 4 > INT32_MAX) return QB_ERR_INVALID;
  return qb_launch_ex(prefill_fp8_join_kernel, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, st, 1, true, p);
}
