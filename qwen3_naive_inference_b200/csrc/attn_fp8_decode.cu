// Single-token attention over the 8-bit paged KV cache (kv_fp8.cuh), plain and grouped.
//
//   o = sum_j p_j vs_j V_j,   p = softmax_j(scale * ks_j * q . K_j)
//
// K_j, V_j the e4m3 codes of key j, ks_j, vs_j the scales of its block of 64 tokens and head.  Every
// key's 256 bytes of codes are read once and meet hq / hkv query rows (a group's members times that),
// so the bound is HBM: 2 * (128 + 1/16) bytes a key and kv head.
//
// A CTA takes one kv head of one sequence (or of a group's shared prefix) and a range of its keys; where there
// are groups enough, one of several members and all their keys (decode_whole_fp8_kernel).  A
// producer warp brings 64-key tiles (8 KB of K, 8 KB of V: one block's codes lie in a row) by TMA into a
// ring of stages; four warps take 16 keys of every tile each and never wait for one another: each keeps
// its own running reference, sum and output, joined once at the end.
//   S^T = K Q^T    mma m16n8k16: the 16 keys are the M rows, up to eight query rows the N columns.  Codes
//                  become halves exactly (cvt); q is scaled by a power of two per row, so that its bf16
//                  value is a half's too.  ks and the softmax scale meet the fp32 sums.
//   P           =  2^(x - ref), halves.  ref follows the largest score so far minus 7 and moves only when
//                  a score passes it by 15: P stays below 2^15 and loses nothing above 2^-31 of the largest.
//   O^T += vs V^T P^T   the 128 head elements are the M rows (8 tiles), the warp's 16 keys the K dimension,
//                  so a tile's product is one mma per 16 elements: vs, one number a tile, joins with the
//                  fp32 accumulator.
// Where a CTA's tiles have scales over 16 times its first one's, or under a 16th, a probability that is nothing beside
// the largest may still make the output (and near the ends of the exponent range vs P V leaves it).  The producer,
// which has the scales in hand, sees it; the CTA then writes nothing and takes a second pass, which weighs before it
// rounds: P = 2^(x + log2 vs - oref), where oref follows the largest x + log2 vs as ref does x, O counts in units of
// 2^oref, and the sum takes sum(P) 2^(oref - log2 vs - ref).  That form for all CTAs cost 10% (512 sequences of up to
// 1024 keys 98 -> 109 us), a choice between the two inside the loop 3%; the second pass costs calls that do not take
// it nothing (plain) to 2% (16 groups of 8, 32 over 4 heads 25.6 -> 26.1; 64 groups, 16 over 8 heads 82.9 -> 83.4).
// The order of head elements and keys inside a product is free, so every operand comes straight from
// 16-byte shared-memory reads (conflict-free under the TMA swizzle) without a transpose but for the
// byte pairs of V (prmt) and P (movmatrix).
// Keys past the range count neither in P (their scores are -inf) nor through V (their codes are zeroed,
// NaN codes of a recycled page included).  Pages outside the pool are reported and their tile skipped.
//
// Measured on a B200 (16 query and 8 kv heads, 128 elements; a plain copy reaches 6.52 TB/s):
//   512 sequences of 64 to 1024 keys      98 us, 556 MB: 5.7 TB/s (one state again and again; 101 to 107, by box, where
//                                         the caches change from call to call: 5.2 to 5.5)
//   16 sequences of 2048 to 32768 keys      88 us, 458 MB: 5.2 TB/s (ragged lengths: CTAs end at different times);
//                                         as many bytes in equal lengths: 6.5 TB/s and more
//   one sequence of 700 keys              8.6 us: the chain of lookups (length, page, scale), copy and join
//   64 groups of 8, 64 to 512 shared and 170 to 512 own keys   83 us, 404 MB: 4.9 TB/s (84 to 86 where the caches change)
//   16 groups of 8, 87 to 700 shared and 100 to 300 own keys   40 over 8 heads 40 us, 70 MB; 32 over 4 heads 26 us, 35 MB:
//                                         a quarter and a fifth of HBM; with five heads and more a kv head a CTA takes one
//                                         member, so each streams the shared keys for itself, from L2 if not from HBM
// What a CTA needs before its first and after its last tile is as long as two to four tiles, and three CTAs of an
// SM hide it only in part: 4096 CTAs of one key each take 21 us.  Longer work a CTA (decode_whole_fp8_kernel) pays
// where members share it, not for plain sequences of these lengths (512 of up to 750 keys: 86 us against 80).
// Fewer warps a CTA and more CTAs an SM (two warps, four to six CTAs: 110 to 120 us for the 512 sequences), three
// stages and four CTAs (111), CTAs that live on and take sequence after sequence (127) or equal shares of all
// keys (133) were slower.
#include <float.h>

#include "attn_fp8.cuh"

namespace {

constexpr int DC_WARPS = 4, DC_THREADS = DC_WARPS * 32 + 32;  // consumers, producer
constexpr int DC_STAGES = 4;
constexpr int DC_STAGE_BYTES = 2 * KV8_TILE;       // K then V
constexpr int DC_MAX_TILES = 128;                  // of one CTA's range (8192 keys)
constexpr int DC_WS_ROW = KV8_D + 4;               // workspace row: O / l, then ref + log2 l
constexpr int DC_O_ROW = KV8_D + 4;                // shared-memory row of a warp's output (padded)
constexpr int DC_META = DC_MAX_TILES * 16 + (2 * DC_STAGES + 1) * 8 + 8 + (3 * DC_WARPS * 16 + 2) * 4;
constexpr int DC_MOST = (2 * DC_STAGES + 2) * 8 + DC_MAX_TILES * 16 + 3 * DC_WARPS * 16 * 4;  // where `most_of` lies in it
constexpr int DC_LEFT = DC_MOST + 4;  // set where a work's scales were far apart
constexpr int DC_SMEM = DC_STAGES * DC_STAGE_BYTES + DC_META + 1024 /*align*/;
static_assert(DC_WARPS * 16 * DC_O_ROW * 4 <= DC_STAGES * DC_STAGE_BYTES, "the join reuses the stages");
constexpr float DC_HEAD = 7.f, DC_SLACK = 15.f;    // ref = max - 7; moves when a score is above ref + 15
// How far a CTA's scales may be from its first tile's, and the range of that, without weighing before rounding: a P
// that is lost (2^-32 of the largest) is then at most 2^-24 of the output's largest share, and |O| below
// 2^15 * 448 * 8192 * 16 vs.
constexpr float DC_NEAR = 16.f, DC_VS_LEAST = 0x1p-100f, DC_VS_MOST = 0x1p60f;
// Weighed, a tile whose scale is less than 2^-50 of the largest (a block of zeros under the smallest scale, say) may
// hold probability although its P, as small as 2^-126, does not: its sum is taken from 2^(x - ref).  Within 2^50
// a P below 2^-100 has x - ref below -42: with x', vs' of the key that set oref, oref is at most x' + log2 vs' - 7,
// and x' at most ref + 15.
constexpr float DC_APART = 0x1p-50f;

struct DecodeP {
  const bf16* q;
  int64_t q_stride;
  const float* ks;
  const float* vs;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_width;
  const int32_t* seqlens;
  int seqlen_add;
  int batch, hq, hkv;
  float scale_log2;
  int own_tokens, own_splits, n_slots;
  float* ws;
  bf16* out;
  int* err;
  // grouped
  const int32_t* members;     // [n_groups, 8], -1 padded
  const int32_t* shared_len;
  const int32_t* kv_start;
  int n_groups, shared_tokens, shared_splits;
  int chunk, n_chunks;        // members per shared CTA, shared CTAs per group
  int group_step;             // shared CTA r takes groups r, r + group_step, ...
  unsigned n_shared;          // shared CTAs; the own CTAs follow
  int* entry_of;              // [batch] in the workspace: where a sequence stands in `members`
};

// The cache's tensor maps: whole blocks, and 16 rows for the blocks that a range ends in.
struct DecodeMaps {
  CUtensorMap k, v, k16, v16;
};
bool decode_maps(DecodeMaps* m, const void* k, const void* v, int64_t num_blocks, int hkv) {
  return kv8_tmap(&m->k, k, num_blocks, hkv, KV8_BLOCK) && kv8_tmap(&m->v, v, num_blocks, hkv, KV8_BLOCK) &&
         kv8_tmap(&m->k16, k, num_blocks, hkv, 16) && kv8_tmap(&m->v16, v, num_blocks, hkv, 16);
}

// What a CTA works on: `rows` query rows over keys [begin, end) of table row `table`.
struct Work {
  int rows, table, begin, end, slot;  // slot: of the workspace, -1: straight to the output
};

QB_DEVICE void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
QB_DEVICE uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
QB_DEVICE uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
QB_DEVICE uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
QB_DEVICE float dc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Row r of a CTA's work: its sequence and head, or -1.
template <bool SHARED>
QB_DEVICE int row_sequence(const DecodeP& p, const int32_t* members, int b, int r) {
  if (!SHARED) return b;
  const int m = members[r / (p.hq / p.hkv)];
  return m >= 0 && m < p.batch ? m : -1;
}

// A sequence's own keys are [first, len); first is a block's start (-1: it is not).
QB_DEVICE int own_first(const DecodeP& p, int b) {
  const int first = p.kv_start ? p.kv_start[b] : 0;
  return first >= 0 && first % KV8_BLOCK == 0 ? first : -1;
}
// The producer's lanes look up the pages of tiles lane, lane + 32, ... of `tiles` from key `begin` (-1: none).
// No length is needed for it, so it goes ahead while those are on their way.
constexpr int DC_LANE_TILES = DC_MAX_TILES / 32;
QB_DEVICE void find_pages(const DecodeP& p, int table, int64_t begin, int tiles, int (&pages)[DC_LANE_TILES]) {
  if (threadIdx.x < DC_WARPS * 32) return;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < DC_LANE_TILES; ++j) {
    const int64_t col = (begin / KV8_BLOCK + lane + 32 * j) / KV8_SUBS;
    pages[j] = lane + 32 * j < tiles && col < p.bt_width ? p.bt[(int64_t)table * p.bt_stride + col] : -1;
  }
}

// The scores x of a tile into P (pb, B fragments), with the running references, sums and outputs moved along.
template <int NT>
QB_DEVICE void plain_tile(const float (&x)[NT][4], float (&ref)[NT][2], float (&l)[NT][2], float (&o)[NT][8][4],
                          uint32_t (&pb)[NT][2]) {
  bool far = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    far |= fmaxf(x[nt][0], x[nt][2]) > ref[nt][0] + DC_SLACK || fmaxf(x[nt][1], x[nt][3]) > ref[nt][1] + DC_SLACK;
  if (__any_sync(0xffffffffu, far)) {  // the first tile, then rarely: move the reference, scale what is there
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(x[nt][c], x[nt][c + 2]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (m > ref[nt][c] + DC_SLACK) {
          const float now = m - DC_HEAD, alpha = dc_exp2(ref[nt][c] - now);
          ref[nt][c] = now;
          l[nt][c] *= alpha;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            o[nt][k][c] *= alpha;
            o[nt][k][c + 2] *= alpha;
          }
        }
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float r0 = ref[nt][0] == -INFINITY ? 0.f : ref[nt][0], r1 = ref[nt][1] == -INFINITY ? 0.f : ref[nt][1];
    const float p0 = dc_exp2(x[nt][0] - r0), p1 = dc_exp2(x[nt][1] - r1);
    const float p2 = dc_exp2(x[nt][2] - r0), p3 = dc_exp2(x[nt][3] - r1);
    l[nt][0] += p0 + p2;
    l[nt][1] += p1 + p3;
    pb[nt][0] = movmatrix_trans(pack_half2(p0, p1));
    pb[nt][1] = movmatrix_trans(pack_half2(p2, p3));
  }
}
// The same with P weighed by the tile's scale before it is rounded; `orefs`: the warp's references of O, by row.
template <int NT>
QB_DEVICE void weigh_tile(const float (&x)[NT][4], float vs, float most, float* orefs, float (&ref)[NT][2],
                          float (&l)[NT][2], float (&o)[NT][8][4], uint32_t (&pb)[NT][2]) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  const float lvs = log2f(vs);
  const bool apart = vs < most * DC_APART || vs == 0.f;  // the same for the whole warp
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float y[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = fmaxf(x[nt][c], x[nt][c + 2]), at = orefs[8 * nt + 2 * t + c];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      if (m > ref[nt][c] + DC_SLACK) {
        l[nt][c] *= dc_exp2(ref[nt][c] - (m - DC_HEAD));
        ref[nt][c] = m - DC_HEAD;
      }
      if (m + lvs > at + DC_SLACK) {
        const float now = m + lvs - DC_HEAD, alpha = dc_exp2(at - now);
        at = now;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          o[nt][k][c] *= alpha;
          o[nt][k][c + 2] *= alpha;
        }
      }
      __syncwarp();
      if (g == 0) orefs[8 * nt + 2 * t + c] = at;
      // (`at` is -inf where no score, or none with a scale, has come: P is zero all the same)
      const float r = (at == -INFINITY ? 0.f : at) - lvs, lr = ref[nt][c] == -INFINITY ? 0.f : ref[nt][c];
      y[c] = dc_exp2(x[nt][c] - r);
      y[c + 2] = dc_exp2(x[nt][c + 2] - r);
      if (apart) l[nt][c] += dc_exp2(x[nt][c] - lr) + dc_exp2(x[nt][c + 2] - lr);
      else l[nt][c] = fmaf(y[c] + y[c + 2], at == -INFINITY ? 0.f : dc_exp2(r - lr), l[nt][c]);
    }
    pb[nt][0] = movmatrix_trans(pack_half2(y[0], y[1]));
    pb[nt][1] = movmatrix_trans(pack_half2(y[2], y[3]));
  }
  __syncwarp();
}

// Four elements of a row from the warps' outputs `so`, in units of 2^oref, and the row's sum in units of 2^m.
QB_DEVICE float4 join_weighed(const float* so, const float* orefs, float m, float sum) {
  float top = -INFINITY;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < DC_WARPS; ++k) top = fmaxf(top, orefs[k * 16]);
  for (int k = 0; k < DC_WARPS; ++k) {
    const float at = orefs[k * 16], f = at == -INFINITY ? 0.f : exp2f(at - top);
    const float4 x = *reinterpret_cast<const float4*>(so + k * 16 * DC_O_ROW);
    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
  }
  // 2^(top - m) / sum in two factors: value scales reach both ends of the exponent range
  const float units = top == -INFINITY ? 0.f : top - m, half = rintf(0.5f * units), back = exp2f(half);
  const float inv = sum == 0.f ? 0.f : exp2f(units - half) / sum;
  return make_float4(acc.x * inv * back, acc.y * inv * back, acc.z * inv * back, acc.w * inv * back);
}

// One CTA: the work `w` of kv head `kvh`; NT tiles of eight query rows.  `members`: the chunk's member
// list (shared work), `b`: the sequence (own work).  `u0` tiles and `item` works came before in this CTA.
// Nothing is written of work whose scales are far apart (for WEIGH: are not), which `*most_of` says.  Returns the tiles.
template <int NT, bool SHARED, bool WHOLE, bool WEIGH>
QB_DEVICE int decode_work(const DecodeP& p, const DecodeMaps& maps, const int (&pages)[DC_LANE_TILES], uint8_t* smem,
                          uint32_t base, const Work& w, int kvh, const int32_t* members, int b, int u0, int item) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  int n = (w.end - w.begin + KV8_BLOCK - 1) / KV8_BLOCK;
  const int group = p.hq / p.hkv;
  uint8_t* meta = smem + DC_STAGES * DC_STAGE_BYTES;
  const uint32_t bar = base + DC_STAGES * DC_STAGE_BYTES;  // full[S], empty[S], meta
  auto full = [&](int s) { return bar + 8 * s; };
  auto empty = [&](int s) { return bar + 8 * (DC_STAGES + s); };
  const uint32_t ready = bar + 8 * (2 * DC_STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(meta + 8 * (2 * DC_STAGES + 1));
  int* n_of = reinterpret_cast<int*>(meta + 8 * (2 * DC_STAGES + 1) + 4);  // WHOLE: tiles
  int* block_of = reinterpret_cast<int*>(meta + 8 * (2 * DC_STAGES + 2));  // of a tile: (page, head, block), -1: no page
  int* part_of = block_of + DC_MAX_TILES;  // WHOLE: its keys, first row << 8, one past its last row << 16
  float* ks_of = reinterpret_cast<float*>(part_of + DC_MAX_TILES);
  float* vs_of = ks_of + DC_MAX_TILES;
  float* join = vs_of + DC_MAX_TILES;  // [warp][16] ref, [warp][16] l
  float* oref = join + 2 * DC_WARPS * 16;  // [warp][16], WEIGH
  float* most_of = oref + DC_WARPS * 16;   // 0, or not (WEIGH: the largest scale) where the scales are far apart
  int* left_of = reinterpret_cast<int*>(most_of + 1);

  if (warp == DC_WARPS) {
    // ------------------------------------------------------------ producer
    float ks[DC_LANE_TILES], vs[DC_LANE_TILES];
    auto found = [&](int j, int page, int blk) {  // tile lane + 32 j is block `blk` of a sequence, in `page`
      int at = -1;
      if (page < 0 || page >= p.num_blocks) {
        qb_set_err(p.err, QB_DEVERR_PAGE);
      } else {
        at = (page * p.hkv + kvh) * KV8_SUBS + blk % KV8_SUBS;
        ks[j] = p.ks[at];
        vs[j] = p.vs[at];
      }
      block_of[lane + 32 * j] = at;
    };
    if (WHOLE) {
      // the group's shared keys, [0, w.end) of table row w.table, then each member's own, which lane m looks up
      int seq = -1, first = 0, keys = 0;
      if (lane < w.rows / group) {
        seq = members[lane];
        if (seq < 0 || seq >= p.batch) {
          seq = -1;
        } else {
          first = own_first(p, seq);
          keys = p.seqlens[seq] + p.seqlen_add - first;
          if (first < 0 || keys > p.own_tokens) qb_set_err(p.err, QB_DEVERR_SHAPE);
          keys = first < 0 ? 0 : max(0, min(keys, p.own_tokens));
        }
      }
      int last = (keys + KV8_BLOCK - 1) / KV8_BLOCK;  // tile after the member's last, counted from the first own one
      for (int o = 1; o < 8; o *= 2) {
        const int before = __shfl_up_sync(0xffffffffu, last, o);
        if (lane >= o && lane < 8) last += before;
      }
      const int shared = n;
      n += __shfl_sync(0xffffffffu, last, 7);
#pragma unroll
      for (int j = 0; j < DC_LANE_TILES; ++j) {
        const int i = lane + 32 * j, own = i - shared;
        int m = 0;
        for (int k = 0; k < 7; ++k) m += own >= __shfl_sync(0xffffffffu, last, k);
        const int from = __shfl_sync(0xffffffffu, first, m), mine = __shfl_sync(0xffffffffu, keys, m);
        const int to = __shfl_sync(0xffffffffu, last, m), table = __shfl_sync(0xffffffffu, seq, m);
        ks[j] = vs[j] = 0.f;
        if (i >= n) continue;
        const int nth = own - (to - (mine + KV8_BLOCK - 1) / KV8_BLOCK);  // the tile among the member's
        const int blk = own < 0 ? i : from / KV8_BLOCK + nth, row = own < 0 ? w.table : table;
        const int live = own < 0 ? w.end - i * KV8_BLOCK : mine - nth * KV8_BLOCK, col = blk / KV8_SUBS;
        part_of[i] = min(live, KV8_BLOCK) | (own < 0 ? w.rows << 16 : (m * group) << 8 | ((m + 1) * group) << 16);
        found(j, col < p.bt_width ? p.bt[(int64_t)row * p.bt_stride + col] : -1, blk);
      }
      if (lane == 0) *n_of = n;
    } else {
#pragma unroll
      for (int j = 0; j < DC_LANE_TILES; ++j) {
        ks[j] = vs[j] = 0.f;
        if (lane + 32 * j < n) found(j, pages[j], w.begin / KV8_BLOCK + lane + 32 * j);
      }
    }
    __syncwarp();
    auto issue = [&](int i) {
      const int s = (u0 + i) % DC_STAGES, block = block_of[i];
      if (block < 0) {
        mbar_arrive(full(s));
        return;
      }
      const int row = block * KV8_BLOCK;
      const uint32_t at = base + s * DC_STAGE_BYTES;
      const int keys = WHOLE ? part_of[i] & 255 : w.end - w.begin - i * KV8_BLOCK;
      const int parts = (min(keys, KV8_BLOCK) + 15) / 16;  // of 16 keys, the last ones ragged
      mbar_expect_tx(full(s), parts * 2 * 16 * KV8_D);
      if (parts == KV8_BLOCK / 16) {
        tma_load_2d(at, &maps.k, 0, row, full(s));
        tma_load_2d(at + KV8_TILE, &maps.v, 0, row, full(s));
      } else {
        for (int k = 0; k < parts; ++k) {
          tma_load_2d(at + k * 16 * KV8_D, &maps.k16, 0, row + 16 * k, full(s));
          tma_load_2d(at + KV8_TILE + k * 16 * KV8_D, &maps.v16, 0, row + 16 * k, full(s));
        }
      }
    };
    int issued = 0;
    auto issue_to = [&](int last) {
      for (; issued < last; ++issued) {
        const int u = u0 + issued;
        if (u >= DC_STAGES && !mbar_wait(empty(u % DC_STAGES), (uint32_t)(u / DC_STAGES - 1) & 1u, abort_flag, p.err)) break;
        issue(issued);
      }
    };
    if (lane == 0) issue_to(min(n, DC_STAGES));
#pragma unroll
    for (int j = 0; j < DC_LANE_TILES; ++j)
      if (lane + 32 * j < n) {
        ks_of[lane + 32 * j] = ks[j];
        vs_of[lane + 32 * j] = vs[j];
      }
    __syncwarp();
    // Are the scales far apart?  Both passes ask the same way.
    auto look = [&] {
      const float v0 = __shfl_sync(0xffffffffu, vs[0], 0), up = v0 * DC_NEAR, down = v0 / DC_NEAR;
      bool far = v0 < DC_VS_LEAST || v0 > DC_VS_MOST;
#pragma unroll
      for (int j = 0; j < DC_LANE_TILES; ++j) far |= lane + 32 * j < n && (vs[j] > up || vs[j] < down);
      return __any_sync(0xffffffffu, far) && n > 0;
    };
    if (WEIGH) {
      float most = FLT_MIN;  // (scales may all be zero)
#pragma unroll
      for (int j = 0; j < DC_LANE_TILES; ++j) most = fmaxf(most, vs[j]);
      most = warp_max(most);
      const bool far = look();
      if (lane == 0) *most_of = far ? most : 0.f;
    }
    if (lane == 0) mbar_arrive(ready);
    if (!WEIGH) {  // off the way to the first tile
      const bool far = look();
      if (lane == 0) *most_of = far ? 1.f : 0.f;
      if (lane == 0 && far) *left_of = 1;
    }
    if (lane == 0) {
      issue_to(n);
      // never leave with a copy in flight into this CTA's shared memory
      for (int i = max(0, issued - DC_STAGES); i < issued; ++i)
        mbar_drain(full((u0 + i) % DC_STAGES), (uint32_t)((u0 + i) / DC_STAGES) & 1u);
    }
    __syncwarp();
    __syncthreads();
    __syncthreads();
    return n;
  }
  // -------------------------------------------------------------- consumers
  // Q as B fragments: column g of tile nt is row nt * 8 + g; lane t holds elements 32t .. 32t+31, the two
  // halves of product kk (chunk kk / 4, word kk % 4 of the codes' 16-byte chunks) at 32t + 4kk.
  uint32_t qf[NT][8][2];
  float fac[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g;
    const int s = r < w.rows ? row_sequence<SHARED>(p, members, b, r) : -1;
    uint4 raw[4];
    __nv_bfloat162 most = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if (s >= 0)
        raw[i] = reinterpret_cast<const uint4*>(p.q + (int64_t)s * p.q_stride + (kvh * group + r % group) * KV8_D +
                                                32 * t)[i];
      const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) most = __hmax2(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[k])));
    }
    float top = fmaxf(__low2float(most), __high2float(most));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the row's largest value goes to [2^9, 2^10): a bf16 value is a half down to 2^-23 of it
    const int e = max((int)(__float_as_uint(top) >> 23), 10);
    const float mul = __uint_as_float((uint32_t)(263 - e) << 23);
    const float back = __uint_as_float((uint32_t)(e - 9) << 23) * p.scale_log2;
    fac[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);      // rows 2t and 2t + 1 of the tile
    fac[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = mul2(unpack_bf16x2(u[k]), make_float2(mul, mul));
        qf[nt][2 * i + k / 2][k & 1] = pack_half2(f.x, f.y);
      }
    }
  }
  float o[NT][8][4], ref[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    ref[nt][0] = ref[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  }
  bool ok = __all_sync(0xffffffffu, mbar_wait(ready, (uint32_t)item & 1u, abort_flag, p.err));
  if (WHOLE) n = *n_of;
  if (WEIGH) {
    if (lane < 16) oref[warp * 16 + lane] = -INFINITY;
    __syncwarp();
  }
  for (int i = 0; ok && i < n; ++i) {
    const int s = (u0 + i) % DC_STAGES;
    if (!__all_sync(0xffffffffu, mbar_wait(full(s), (uint32_t)((u0 + i) / DC_STAGES) & 1u, abort_flag, p.err))) {
      ok = false;
      break;
    }
    // keys of the tile that count, and for which of the rows
    const int part = WHOLE ? part_of[i] : 0, live = block_of[i] < 0 ? 0 : WHOLE ? part & 255 : w.end - w.begin - i * KV8_BLOCK;
    bool counts[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * nt + 2 * t + c;
        counts[nt][c] = !WHOLE || (r >= ((part >> 8) & 255) && r < part >> 16);
      }
    if (live > 16 * warp) {
      const uint32_t kt = base + s * DC_STAGE_BYTES, vt = kt + KV8_TILE;
      // V^T, asked for first: lane (g, t) holds elements 16g .. 16g+15 of keys 2t, 2t+1, 2t+8, 2t+9
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = 16 * warp + 2 * t + (k & 1) + 8 * (k >> 1);
        v[k] = lds128(vt + row * KV8_D + ((uint32_t)(g ^ ((2 * t + (k & 1)) & 7)) << 4));
        if (live < KV8_BLOCK && row >= live) v[k] = make_uint4(0, 0, 0, 0);
      }
      const uint32_t vw[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                 {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
      float x[NT][4];
      {  // scores of keys 16 warp + g and + 8
        float part[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) part[nt][c][0] = part[nt][c][1] = part[nt][c][2] = part[nt][c][3] = 0.f;
        const uint32_t row = kt + (16 * warp + g) * KV8_D;
        uint4 k0[2], k1[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t off = (uint32_t)((2 * t + c) ^ g) << 4;
          k0[c] = lds128(row + off);
          k1[c] = lds128(row + 8 * KV8_D + off);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t u0[4] = {k0[c].x, k0[c].y, k0[c].z, k0[c].w}, u1[4] = {k1[c].x, k1[c].y, k1[c].z, k1[c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t a[4];
            e4m3x4_to_half2x2(u0[k], a[0], a[2]);
            e4m3x4_to_half2x2(u1[k], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16_16816(part[nt][c], a, qf[nt][4 * c + k][0], qf[nt][4 * c + k][1]);
          }
        }
        const float ks = ks_of[i];
        const bool in0 = 16 * warp + g < live, in1 = 16 * warp + g + 8 < live;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          x[nt][0] = in0 && counts[nt][0] ? (part[nt][0][0] + part[nt][1][0]) * (fac[nt][0] * ks) : -INFINITY;
          x[nt][1] = in0 && counts[nt][1] ? (part[nt][0][1] + part[nt][1][1]) * (fac[nt][1] * ks) : -INFINITY;
          x[nt][2] = in1 && counts[nt][0] ? (part[nt][0][2] + part[nt][1][2]) * (fac[nt][0] * ks) : -INFINITY;
          x[nt][3] = in1 && counts[nt][1] ? (part[nt][0][3] + part[nt][1][3]) * (fac[nt][1] * ks) : -INFINITY;
        }
      }
      // V's fragments do not wait for the scores: they are made while those are on their way
      uint32_t va[8][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t lo = __byte_perm(vw[0][k], vw[1][k], half ? 0x7362 : 0x5140);
          const uint32_t hi = __byte_perm(vw[2][k], vw[3][k], half ? 0x7362 : 0x5140);
          e4m3x4_to_half2x2(lo, va[2 * k + half][0], va[2 * k + half][1]);
          e4m3x4_to_half2x2(hi, va[2 * k + half][2], va[2 * k + half][3]);
        }
      uint32_t pb[NT][2];
      if (WEIGH)
        weigh_tile<NT>(x, vs_of[i], *most_of, oref + warp * 16, ref, l, o, pb);
      else
        plain_tile<NT>(x, ref, l, o, pb);
      const float vs = WEIGH ? 1.f : vs_of[i];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16_16816(d, va[k], pb[nt][0], pb[nt][1]);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (counts[nt][c & 1]) o[nt][k][c] = fmaf(vs, d[c], o[nt][k][c]);  // (else V may be NaN, and P 0)
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty(s));
  }
  // -------------------------------------------------------------- join the four warps
  __syncthreads();  // the producer has drained its copies: the stages are free
  float* so = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nt * 8 + 2 * t + c;
      float sum = l[nt][c];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (r >= w.rows) continue;
      if (g == 0) {
        join[warp * 16 + r] = ref[nt][c];
        join[(DC_WARPS + warp) * 16 + r] = sum;
      }
      float4* dst = reinterpret_cast<float4*>(so + (warp * 16 + r) * DC_O_ROW + 16 * g);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        dst[k] = make_float4(o[nt][2 * k][c], o[nt][2 * k][c + 2], o[nt][2 * k + 1][c], o[nt][2 * k + 1][c + 2]);
    }
  __syncthreads();
  if (*abort_flag || (*most_of > 0.f) != WEIGH) return n;
  for (int i = tid; i < w.rows * 32; i += DC_WARPS * 32) {
    const int r = i >> 5, d = (i & 31) * 4;
    const int seq = row_sequence<SHARED>(p, members, b, r);
    float m = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < DC_WARPS; ++k) m = fmaxf(m, join[k * 16 + r]);
#pragma unroll
    for (int k = 0; k < DC_WARPS; ++k) {
      const float rk = join[k * 16 + r];
      const float f = rk == -INFINITY ? 0.f : exp2f(rk - m);
      const float4 x = *reinterpret_cast<const float4*>(so + (k * 16 + r) * DC_O_ROW + d);
      sum += f * join[(DC_WARPS + k) * 16 + r];
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    if (seq < 0) continue;
    if (WEIGH) {
      acc = join_weighed(so + r * DC_O_ROW + d, oref + r, m, sum);
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    }
    const int64_t row = (int64_t)seq * p.hq + kvh * group + r % group;
    if (w.slot < 0) {
      uint2 u;
      u.x = pack_bf16x2(acc.x, acc.y);
      u.y = pack_bf16x2(acc.z, acc.w);
      *reinterpret_cast<uint2*>(p.out + row * KV8_D + d) = u;
    } else {
      float* ws = p.ws + (row * p.n_slots + w.slot) * DC_WS_ROW;
      *reinterpret_cast<float4*>(ws + d) = acc;
      if (d == 0) ws[KV8_D] = sum == 0.f ? -INFINITY : m + log2f(sum);
    }
  }
  return n;
}

// The splits of a sequence's own keys that hold any.
QB_DEVICE int own_live(const DecodeP& p, int b) {
  const int first = own_first(p, b), keys = p.seqlens[b] + p.seqlen_add - first;
  return first < 0 || keys <= 0 ? 0 : min(p.own_splits, (keys + p.own_tokens - 1) / p.own_tokens);
}

// The CTA's barriers.
QB_DEVICE void decode_barriers(const DecodeMaps& maps, uint8_t* smem, uint32_t base) {
  if (threadIdx.x == 0) {
    const uint32_t bar = base + DC_STAGES * DC_STAGE_BYTES;
    for (int s = 0; s < DC_STAGES; ++s) {
      mbar_init(bar + 8 * s, 1);
      mbar_init(bar + 8 * (DC_STAGES + s), DC_WARPS);
    }
    mbar_init(bar + 16 * DC_STAGES, 1);
    *reinterpret_cast<volatile int*>(smem + DC_STAGES * DC_STAGE_BYTES + 8 * (2 * DC_STAGES + 1)) = 0;
    *reinterpret_cast<int*>(smem + DC_STAGES * DC_STAGE_BYTES + DC_LEFT) = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.v)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.k16)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.v16)) : "memory");
  }
  __syncthreads();
}
// The barriers of a pass that is done may be made anew.
QB_DEVICE void barriers_back(uint8_t* smem, uint32_t base) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 0; i < 2 * DC_STAGES + 1; ++i)
      asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(base + DC_STAGES * DC_STAGE_BYTES + 8 * i) : "memory");
}
// The stages, which a join wrote to, go back to the copies.
QB_DEVICE void stages_back() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
}

// Did the pass leave work to the one that weighs?
QB_DEVICE bool left_to_weigh(const uint8_t* smem) {
  const uint8_t* meta = smem + DC_STAGES * DC_STAGE_BYTES;
  const bool aborted = *reinterpret_cast<const volatile int*>(meta + 8 * (2 * DC_STAGES + 1)) != 0;
  return !aborted && *reinterpret_cast<const int*>(meta + DC_LEFT) != 0;
}

// The CTA's work, or (WEIGH) what the pass before left of it; true if some was left.  NTS, NTO: row tiles of a shared
// and of an own CTA (NTS = 0: no groups).
template <int NTS, int NTO, bool WEIGH>
QB_DEVICE bool decode_pass(const DecodeMaps& maps, const DecodeP& p, uint8_t* smem, uint32_t base) {
  unsigned i = blockIdx.x;
  const int group = p.hq / p.hkv;
  int pages[DC_LANE_TILES];
  if (NTS > 0 && i < p.n_shared) {
    const int split = i % p.shared_splits;
    i /= p.shared_splits;
    const int kvh = i % p.hkv;
    i /= p.hkv;
    const int c = i % p.n_chunks, first = i / p.n_chunks;
    int u0 = 0, item = 0;
    for (int grp = first; grp < p.n_groups; grp += p.group_step) {
      const int32_t* members = p.members + grp * 8 + c * p.chunk;
      const int donor = p.members[grp * 8], keys = p.shared_len[grp];
      if (donor >= 0 && donor < p.batch) find_pages(p, donor, split * p.shared_tokens, p.shared_tokens / KV8_BLOCK, pages);
      Work w;
      const int n_members = min(p.chunk, 8 - c * p.chunk);
      w.rows = n_members * group;
      w.table = donor;
      w.begin = split * p.shared_tokens;
      w.end = min(keys, w.begin + p.shared_tokens);
      w.slot = split;
      bool any = false;
      for (int m = 0; m < n_members; ++m) {
        const int b = members[m];
        any |= b >= 0 && b < p.batch;
        if (kvh == 0 && split == 0 && threadIdx.x == 0) {
          if (b >= p.batch) qb_set_err(p.err, QB_DEVERR_SHAPE);
          else if (b >= 0) p.entry_of[b] = grp * 8 + c * p.chunk + m;
        }
      }
      if (split == p.shared_splits - 1 && w.end < keys && threadIdx.x == 0) qb_set_err(p.err, QB_DEVERR_SHAPE);
      if (!any || w.begin >= w.end || donor < 0 || donor >= p.batch) continue;
      if (item > 0) stages_back();
      u0 += decode_work<NTS == 0 ? 1 : NTS, true, false, WEIGH>(p, maps, pages, smem, base, w, kvh, members, 0, u0, item);
      ++item;
    }
    return left_to_weigh(smem);
  }
  i -= p.n_shared;
  const int split = i % p.own_splits;
  i /= p.own_splits;
  const int kvh = i % p.hkv;
  const int b = i / p.hkv;
  const int len = p.seqlens[b] + p.seqlen_add, first = own_first(p, b);
  const int64_t begin = (int64_t)first + (int64_t)split * p.own_tokens;
  find_pages(p, b, max(begin, (int64_t)0), p.own_tokens / KV8_BLOCK, pages);
  if ((first < 0 || (split == p.own_splits - 1 && begin + p.own_tokens < len)) && threadIdx.x == 0)
    qb_set_err(p.err, QB_DEVERR_SHAPE);
  if (first < 0) return false;
  Work w;
  w.rows = group;
  w.table = b;
  w.begin = (int)min(begin, (int64_t)max(len, 0));
  w.end = (int)min((int64_t)max(len, 0), begin + p.own_tokens);
  // a sequence whose keys are all here has nothing to join; with one slot there is no workspace
  w.slot = NTS == 0 && (p.n_slots == 1 || (split == 0 && w.end == len)) ? -1 : (NTS > 0 ? p.shared_splits : 0) + split;
  if (w.begin >= w.end) {
    if (p.n_slots == 1)  // no keys at all
      for (int k = threadIdx.x; k < group * KV8_D / 4; k += DC_THREADS)
        reinterpret_cast<uint2*>(p.out + ((int64_t)b * p.hq + kvh * group) * KV8_D)[k] = make_uint2(0, 0);
    return false;
  }
  decode_work<NTO, false, false, WEIGH>(p, maps, pages, smem, base, w, kvh, nullptr, b, 0, 0);
  return left_to_weigh(smem);
}
template <int NTS, int NTO>
QB_DEVICE void decode_weigh(const DecodeMaps& maps, const DecodeP& p, uint8_t* smem, uint32_t base) {
  barriers_back(smem, base);
  decode_barriers(maps, smem, base);
  decode_pass<NTS, NTO, true>(maps, p, smem, base);
}

template <int NTS, int NTO>
__global__ void __launch_bounds__(DC_THREADS, 3)
decode_fp8_kernel(const __grid_constant__ DecodeMaps maps, const __grid_constant__ DecodeP p) {
  extern __shared__ uint8_t smem_raw[];
  qb_pdl_trigger();
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  decode_barriers(maps, smem, base);
  qb_pdl_wait();
  if (decode_pass<NTS, NTO, false>(maps, p, smem, base)) decode_weigh<NTS, NTO>(maps, p, smem, base);
}

// Whole groups are taken where the longest CTA's keys are no more than this for the number of CTAs: with few CTAs
// its length is the call's, with many its fewer beginnings and ends count.  Measured (us per call, whole / split;
// eight heads, so 16 CTAs a group of eight; the keys a CTA has at most):
//    2 groups, 768 keys 11.3 / 12.7, 1280 keys 13.4 / 13.0, 1792 keys 16.5 / 13.1
//    8 groups, 832 keys 12.9 / 14.6, 1344 keys 18.6 / 18.2, 3328 keys 34 / 27
//   16 groups, 1344 keys 21.9 / 27.6, 1792 keys 25.2 / 29.7, 3328 keys 43 / 39
//   24 groups, 1024 keys 20 / 32, 3328 keys 46 / 54;   64 groups, 1024 keys 41 / 72, 3328 keys 103 / 119
constexpr int DC_WHOLE_KEYS = 512, DC_WHOLE_KEYS_PER_CTA = 8;
// Whole groups: a CTA takes up to eight query rows of a group -- four members, where two query heads share a
// kv head -- through the shared keys and then through each member's own, one after another in the same ring
// and the same running sums; own tiles count for their member's rows only.  Nothing is left to join, and what a
// CTA needs to begin and to end (as long as four tiles of keys take) is paid once for four members.
template <int NT, bool WEIGH>
QB_DEVICE bool decode_whole_pass(const DecodeMaps& maps, const DecodeP& p, uint8_t* smem, uint32_t base) {
  unsigned i = blockIdx.x;
  const int group = p.hq / p.hkv;
  if (i >= p.n_shared) {  // a warp per sequence: zeros for those in no group
    const int64_t b = (int64_t)(i - p.n_shared) * (DC_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (b >= p.batch) return false;
    bool member = false;
    for (int k = lane; k < p.n_groups * 8; k += 32) member |= p.members[k] == (int)b;
    if (__any_sync(0xffffffffu, member)) return false;
    for (int k = lane; k < p.hq * KV8_D / 8; k += 32)
      reinterpret_cast<uint4*>(p.out + b * p.hq * KV8_D)[k] = make_uint4(0, 0, 0, 0);
    return false;
  }
  const int kvh = i % p.hkv;
  i /= p.hkv;
  const int c = i % p.n_chunks, n_members = min(p.chunk, 8 - c * p.chunk);
  int u0 = 0, item = 0, pages[DC_LANE_TILES];
  for (int grp = i / p.n_chunks; grp < p.n_groups; grp += p.group_step) {
    const int32_t* members = p.members + grp * 8 + c * p.chunk;
    const int donor = p.members[grp * 8], keys = p.shared_len[grp];
    bool any = false, wrong = false;
    for (int m = 0; m < n_members; ++m) {
      any |= members[m] >= 0 && members[m] < p.batch;
      wrong |= members[m] >= p.batch;
    }
    if ((wrong || keys > p.shared_tokens) && threadIdx.x == 0) qb_set_err(p.err, QB_DEVERR_SHAPE);
    if (!any) continue;
    Work w;
    w.rows = n_members * group;
    w.table = donor;
    w.begin = 0;
    w.end = donor >= 0 && donor < p.batch ? max(0, min(keys, p.shared_tokens)) : 0;
    w.slot = -1;
    if (item > 0) stages_back();
    u0 += decode_work<NT, true, true, WEIGH>(p, maps, pages, smem, base, w, kvh, members, 0, u0, item);
    ++item;
  }
  return left_to_weigh(smem);
}
template <int NT>
QB_DEVICE void decode_whole_weigh(const DecodeMaps& maps, const DecodeP& p, uint8_t* smem, uint32_t base) {
  barriers_back(smem, base);
  decode_barriers(maps, smem, base);
  decode_whole_pass<NT, true>(maps, p, smem, base);
}

template <int NT>
__global__ void __launch_bounds__(DC_THREADS, 3)
decode_whole_fp8_kernel(const __grid_constant__ DecodeMaps maps, const __grid_constant__ DecodeP p) {
  extern __shared__ uint8_t smem_raw[];
  qb_pdl_trigger();
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  decode_barriers(maps, smem, base);
  qb_pdl_wait();
  if (decode_whole_pass<NT, false>(maps, p, smem, base)) decode_whole_weigh<NT>(maps, p, smem, base);
}

// Joins the splits of a (sequence, head): a warp each, weights 2^(lse - largest lse).  Only the splits
// that hold keys were written and are read.
__global__ void __launch_bounds__(128)
decode_fp8_join_kernel(DecodeP p) {
  qb_pdl_trigger();
  qb_pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int h = (int)(item % p.hq);
  const int b = (int)(item / p.hq);
  if (b >= p.batch) return;
  int n_shared = 0;
  bool member = true;
  if (p.members) {
    // entry_of holds whatever was there for a sequence in no group: it counts where `members` agrees
    const int e = p.entry_of[b];
    member = e >= 0 && e < p.n_groups * 8 && p.members[e] == b;
    if (member) {
      const int donor = p.members[e / 8 * 8], keys = p.shared_len[e / 8];
      if (donor >= 0 && donor < p.batch && keys > 0)
        n_shared = min(p.shared_splits, (keys + p.shared_tokens - 1) / p.shared_tokens);
    }
  }
  const int own0 = p.members ? p.shared_splits : 0, n = member ? n_shared + own_live(p, b) : 0;
  if (!p.members && n == 1) return;  // its only CTA has written the output
  const float* ws = p.ws + ((int64_t)b * p.hq + h) * p.n_slots * DC_WS_ROW;
  auto slot = [&](int s) { return ws + (int64_t)(s < n_shared ? s : own0 + s - n_shared) * DC_WS_ROW; };
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, slot(s)[KV8_D]);
  m = warp_max(m);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float* at = slot(s);
    const float lse = at[KV8_D], f = lse == -INFINITY ? 0.f : exp2f(lse - m);
    const float4 x = *reinterpret_cast<const float4*>(at + lane * 4);
    sum += f;
    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint2 u;
  u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + ((int64_t)b * p.hq + h) * KV8_D + lane * 4) = u;
}

template <int NTS, int NTO>
int launch_decode(const DecodeMaps& maps, const DecodeP& p, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const int may = kv8_allow_smem(reinterpret_cast<const void*>(decode_fp8_kernel<NTS, NTO>), DC_SMEM, allowed);
  if (may != QB_OK) return may;
  const int64_t ctas = p.n_shared + (int64_t)p.batch * p.hkv * p.own_splits, rows = (int64_t)p.batch * p.hq;
  if (ctas > INT32_MAX || rows > INT32_MAX) return QB_ERR_INVALID;
  const int rc = qb_launch_ex(decode_fp8_kernel<NTS, NTO>, dim3((unsigned)ctas), dim3(DC_THREADS), DC_SMEM, st, 1, true,
                              maps, p);
  if (rc != QB_OK || p.n_slots == 1) return rc;
  return qb_launch_ex(decode_fp8_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, 1, true, p);
}

template <int NT>
int launch_whole(const DecodeMaps& maps, const DecodeP& p, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const int may = kv8_allow_smem(reinterpret_cast<const void*>(decode_whole_fp8_kernel<NT>), DC_SMEM, allowed);
  if (may != QB_OK) return may;
  const int64_t ctas = p.n_shared + ((int64_t)p.batch + DC_THREADS / 32 - 1) / (DC_THREADS / 32);
  if (ctas > INT32_MAX) return QB_ERR_INVALID;
  return qb_launch_ex(decode_whole_fp8_kernel<NT>, dim3((unsigned)ctas), dim3(DC_THREADS), DC_SMEM, st, 1, true, maps, p);
}

// floats of the splits' partial outputs
size_t decode_partials(int batch, int hq, int n_slots) { return (size_t)batch * hq * n_slots * DC_WS_ROW; }

int members_per_cta(int group) { return min(8, (group <= 8 ? 8 : 16) / group); }

bool split_ok(int tokens, int splits) {
  return tokens > 0 && tokens % KV8_BLOCK == 0 && tokens <= DC_MAX_TILES * KV8_BLOCK && splits >= 1 &&
         (int64_t)tokens * splits <= INT32_MAX / 2;
}

}  // namespace

extern "C" int qb_paged_decode_attn_fp8(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                                        const float* k_scale, const float* v_scale, int64_t num_blocks, int page_size,
                                        const int32_t* block_tables, int64_t bt_stride, int bt_width,
                                        const int32_t* seqlens, int seqlen_add, int batch, int hq, int hkv, int D,
                                        float scale, int split_tokens, int max_splits, float* workspace, void* out,
                                        int* err, qb_stream_t stream) {
  if (D != KV8_D || page_size != KV8_PAGE) return QB_ERR_UNSUPPORTED;
  QB_CHECK_ARG(batch >= 0 && split_ok(split_tokens, max_splits));
  if (batch == 0) return QB_OK;
  const int ok = kv8_check_cache(q, q_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_tables, bt_stride,
                                 bt_width, hq, hkv, out);
  if (ok != QB_OK) return ok;
  QB_CHECK_ARG(seqlens && (max_splits == 1 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)));
  DecodeMaps maps;
  if (!decode_maps(&maps, k_cache, v_cache, num_blocks, hkv)) return QB_ERR_INVALID;
  DecodeP p{};
  p.q = (const bf16*)q; p.q_stride = q_stride; p.ks = k_scale; p.vs = v_scale; p.num_blocks = num_blocks;
  p.bt = block_tables; p.bt_stride = bt_stride; p.bt_width = bt_width; p.seqlens = seqlens; p.seqlen_add = seqlen_add;
  p.batch = batch; p.hq = hq; p.hkv = hkv; p.scale_log2 = scale * KV8_LOG2E;
  p.own_tokens = split_tokens; p.own_splits = max_splits; p.n_slots = max_splits;
  p.ws = workspace; p.out = (bf16*)out; p.err = err;
  const cudaStream_t st = (cudaStream_t)stream;
  return hq / hkv <= 8 ? launch_decode<0, 1>(maps, p, st) : launch_decode<0, 2>(maps, p, st);
}

extern "C" int qb_paged_decode_grouped_fp8_whole(int hq, int hkv, int group_step, int shared_tokens, int shared_splits,
                                                 int own_tokens, int own_splits) {
  if (shared_splits != 1 || own_splits != 1 || hkv < 1 || hq / hkv < 1 || hq / hkv > KV8_MAX_GROUP) return 0;
  const int chunk = members_per_cta(hq / hkv);
  const int64_t ctas = (int64_t)group_step * ((8 + chunk - 1) / chunk) * hkv;
  const int64_t keys = shared_tokens + (int64_t)chunk * own_tokens;
  return ctas > 0 && keys <= DC_MAX_TILES * KV8_BLOCK && keys <= DC_WHOLE_KEYS + DC_WHOLE_KEYS_PER_CTA * ctas;
}

extern "C" int qb_paged_decode_attn_grouped_fp8(
    const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const float* k_scale,
    const float* v_scale, int64_t num_blocks, int page_size, const int32_t* block_tables, int64_t bt_stride,
    int bt_width, const int32_t* seqlens, int seqlen_add, int batch, int hq, int hkv, int D, float scale,
    const int32_t* group_members, const int32_t* shared_len, int n_groups, const int32_t* kv_start, int group_step,
    int shared_tokens, int shared_splits, int own_tokens, int own_splits, float* workspace, void* out, int* err, qb_stream_t stream) {
  if (D != KV8_D || page_size != KV8_PAGE) return QB_ERR_UNSUPPORTED;
  QB_CHECK_ARG(batch >= 0 && n_groups >= 0 && n_groups <= INT32_MAX / 8 && group_step >= 1 && split_ok(shared_tokens, shared_splits) &&
               split_ok(own_tokens, own_splits) && shared_splits <= INT32_MAX - own_splits);
  if (batch == 0 || n_groups == 0) return QB_OK;
  const int ok = kv8_check_cache(q, q_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_tables, bt_stride,
                                 bt_width, hq, hkv, out);
  if (ok != QB_OK) return ok;
  const bool whole =
      qb_paged_decode_grouped_fp8_whole(hq, hkv, min(group_step, n_groups), shared_tokens, shared_splits, own_tokens, own_splits);
  QB_CHECK_ARG(seqlens && group_members && shared_len && kv_start &&
               (whole || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)));
  DecodeMaps maps;
  if (!decode_maps(&maps, k_cache, v_cache, num_blocks, hkv)) return QB_ERR_INVALID;
  DecodeP p{};
  p.q = (const bf16*)q; p.q_stride = q_stride; p.ks = k_scale; p.vs = v_scale; p.num_blocks = num_blocks;
  p.bt = block_tables; p.bt_stride = bt_stride; p.bt_width = bt_width; p.seqlens = seqlens; p.seqlen_add = seqlen_add;
  p.batch = batch; p.hq = hq; p.hkv = hkv; p.scale_log2 = scale * KV8_LOG2E;
  p.own_tokens = own_tokens; p.own_splits = own_splits; p.n_slots = shared_splits + own_splits;
  p.ws = workspace; p.out = (bf16*)out; p.err = err;
  p.members = group_members; p.shared_len = shared_len; p.kv_start = kv_start; p.n_groups = n_groups;
  p.shared_tokens = shared_tokens; p.shared_splits = shared_splits;
  // Eight query rows a CTA where they are enough for a member: with 16, a group's shared keys were read
  // once instead of twice (the second time from L2), but a CTA's registers spilled and its sixteen rows took
  // longer to join (64 groups of 8: 102 us against 107, five small groups 11.6 against 16.3).
  const int row_tiles = hq / hkv <= 8 ? 1 : 2;
  p.chunk = members_per_cta(hq / hkv);
  p.n_chunks = (8 + p.chunk - 1) / p.chunk;
  p.group_step = min(group_step, n_groups);
  p.entry_of = whole ? nullptr : reinterpret_cast<int*>(workspace + decode_partials(batch, hq, p.n_slots));
  const int64_t shared = (int64_t)p.group_step * p.n_chunks * hkv * shared_splits;
  QB_CHECK_ARG(shared <= INT32_MAX);
  p.n_shared = (unsigned)shared;
  const cudaStream_t st = (cudaStream_t)stream;
  if (whole)
    return row_tiles == 1 ? launch_whole<1>(maps, p, st) : launch_whole<2>(maps, p, st);
  return row_tiles == 1 ? launch_decode<1, 1>(maps, p, st) : launch_decode<2, 2>(maps, p, st);
}

extern "C" size_t qb_paged_decode_fp8_workspace_bytes(int batch, int hq, int n_slots) {
  return n_slots <= 1 ? 0 : decode_partials(batch, hq, n_slots) * 4;
}

extern "C" size_t qb_paged_decode_grouped_fp8_workspace_bytes(int batch, int hq, int n_slots) {
  return decode_partials(batch, hq, n_slots) * 4 + ((size_t)batch * 4 + 15) / 16 * 16;
}
