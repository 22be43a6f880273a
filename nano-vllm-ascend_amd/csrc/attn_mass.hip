// Attention mass: what each cached token is given by the softmax, summed over the query heads of its kv head - the statistic
// that an eviction from the cache goes by (kv_evict.hip).
//
//   decode   o_h = sum_j p_hj v_j, mass_j += sum_h p_hj for one new token per sequence
//   prompt   mass_j += sum_i sum_h p_hij for the last rows of each sequence's prompt
//
// A weight is known only once its row's maximum and sum are, so the scores are needed twice.  Decode keeps them (4 bytes a token
// and query head, beside the 4 * head_dim bytes of K and V that it streams anyway); the prompt form, whose scores are as many
// as its products are long, takes the products twice.  Nothing is added with atomics: a token of a kv head has one writer, and
// the same call gives the same bits.
#include <algorithm>

#include "mi_common.hpp"

namespace mi {
namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4;     // one MFMA 16x16x16 bf16 operand
typedef __attribute__((ext_vector_type(16))) float f32x16;   // one MFMA 32x32 C/D fragment

struct Pages {
  const int32_t* table;
  int64_t table_stride;
  int64_t num_blocks;
  int tpb;        // 16-token tiles per block
  int tpb_shift;  // log2 of it, -1 where it is no power of two
  int cap;        // tokens that a table row has room for
  int n_kv;
};

// an entry of a table, which no kernel here writes: by way of the constant address space a wave-uniform index is a scalar read, also behind stores
__device__ __forceinline__ int32_t entry(const int32_t* row, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(row))[i];
}
__device__ __forceinline__ int block_of(const Pages& pg, int t) { return pg.tpb_shift >= 0 ? t >> pg.tpb_shift : t / pg.tpb; }
// element offset of tile t of kv head h in block blk; `there`: that is a block of the cache (reads go to block 0 otherwise)
template <int D>
__device__ __forceinline__ int64_t tile_in(const Pages& pg, int32_t blk, int t, int h, bool& there) {
  there = blk >= 0 && blk < pg.num_blocks;
  return (((there ? (int64_t)blk : 0) * pg.n_kv + h) * pg.tpb + (t - block_of(pg, t) * pg.tpb)) * (16 * D);
}
template <int D>
__device__ __forceinline__ int64_t tile_at(const Pages& pg, const int32_t* row, int t, int h, bool& there) {
  return tile_in<D>(pg, entry(row, block_of(pg, t)), t, h, there);
}

int tile_shift(int block_size) {
  const int tpb = block_size / 16;
  return (tpb & (tpb - 1)) == 0 ? __builtin_ctz(tpb) : -1;
}

struct MassRows {
  float* mass;            // [rows][n_kv][len]
  int64_t rows, len;
  const int32_t *slots, *slots_out;
  int n_kv;
  __device__ const float* in(int b, int h) const {
    const int64_t r = slots[b];
    return r >= 0 && r < rows ? mass + (r * n_kv + h) * len : nullptr;
  }
  __device__ float* out(int b, int h) const {
    const int64_t r = slots_out[b];
    return r >= 0 && r < rows ? mass + (r * n_kv + h) * len : nullptr;
  }
};

// ---------------------------------------------------------------------------------------------------------------------
// decode
//
// One workgroup of 8 waves per (kv head, split, sequence).  As in the plain decode attention a wave walks a run of 32-token
// chunks with two chunks' K and V requested ahead, S^T = K Q^T and O^T += V^T P on the matrix cores, P as bf16 hi + lo; its
// scores go out in 32 bits on the way (64-byte pieces per head and tile).  The waves join in LDS.  With one split the workgroup
// then reads its scores back (they are in its XCD's L2) and adds the weights; with more a second launch joins the splits, too.
//
// Bound by HBM: 208 us for 8 contexts of 32768 tokens, 64 heads of 128 on 8 (K, V, the scores and the splits' sums, 1.145 GB: 5.5 TB/s) and 18 for
// the join (84 MB), 24 us for 32 x 1024 of 16 heads on 8 (138 MB: 5.7 TB/s), 54 + 8 for one of 131072 of 32 heads of 64 on 8 (285 MB: 5.3 TB/s).
// ---------------------------------------------------------------------------------------------------------------------
struct DecodeMass {
  const uint16_t* q;
  int64_t q_stride;
  const uint16_t *kc, *vc;
  Pages pg;
  const int32_t* lens;
  MassRows rows;
  uint16_t* out;
  float* scores;   // [batch * n_q][cap], log2 domain
  float* part_o;   // [batch * n_q][splits][D]
  float* part_ml;  // [batch * n_q][splits][2]
  int G, splits;
  float scale_log2e;
};

constexpr int DW = 8;             // waves of a decode workgroup
constexpr int MAX_SPLITS = 64;    // one wave joins a head's splits

template <int DB>
struct Chunk {
  u32x4 K[2][DB], V[2][DB];
};

template <int DB>
__global__ __launch_bounds__(DW * 64) void decode_mass_kernel(DecodeMass a) {
  constexpr int D = 32 * DB;
  __shared__ __attribute__((aligned(16))) float sm_o[DW][16][D];
  __shared__ float sm_m[DW][16], sm_l[DW][16], sm_M[16], sm_inv[16];

  const int h = blockIdx.x, split = blockIdx.y, b = blockIdx.z, G = a.G;
  const int ctx = min(max(a.lens[b], 0), a.pg.cap);
  const int n_tiles = (ctx + 15) >> 4, n_chunks = (n_tiles + 1) >> 1, n_waves = DW * a.splits;
  const int deal_q = n_chunks / n_waves, deal_r = n_chunks % n_waves;
  auto deal = [&](int r) { return r * deal_q + min(r, deal_r); };
  const int64_t row0 = (int64_t)b * a.pg.n_kv * G + (int64_t)h * G;
  if (deal(split * DW) >= deal((split + 1) * DW)) {  // nothing here for this split
    if (a.splits == 1) {
      for (int i = threadIdx.x; i < G * (D / 2); i += DW * 64) *reinterpret_cast<uint32_t*>(a.out + row0 * D + 2 * i) = 0u;
    } else if ((int)threadIdx.x < G) {
      float* ml = a.part_ml + ((row0 + threadIdx.x) * a.splits + split) * 2;
      ml[0] = -INFINITY;
      ml[1] = 0.f;
    }
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int32_t* row = a.pg.table + (int64_t)b * a.pg.table_stride;
  const float* const had = a.rows.in(b, h);  // (read here: a dependent read less at the end)
  float* const now = a.rows.out(b, h);
  const int c0 = deal(split * DW + wave), c1 = deal(split * DW + wave + 1);

  bf16x8 Q[DB];
#pragma unroll
  for (int kk = 0; kk < DB; ++kk) {
    u32x4 v = {0, 0, 0, 0};
    if (n < G) v = *reinterpret_cast<const u32x4*>(a.q + b * a.q_stride + (int64_t)(h * G + n) * D + 8 * g + 32 * kk);
    Q[kk] = as_frag(v);
  }
  float m = -INFINITY, l = 0.f;
  f32x4 acc[2 * DB];
#pragma unroll
  for (int j = 0; j < 2 * DB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float* const score_row = a.scores + (row0 + n) * (int64_t)a.pg.cap;

  // a chunk's second tile may be behind the context: the first one again, masked
  auto load = [&](int c, Chunk<DB>& x) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bool there;
      const int64_t at = tile_at<D>(a.pg, row, min(2 * c + i, n_tiles - 1), h, there);
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) x.K[i][kk] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.kc + at + kk * 512 + lane * 8));
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) x.V[i][kk] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.vc + at + kk * 512 + lane * 8));
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto attend = [&](int c, Chunk<DB>& x) __attribute__((always_inline)) {
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int kk = 0; kk < DB; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_frag(x.K[i][kk]), Q[kk], s[i], 0, 0, 0);
    bool there0, there1;
    tile_at<D>(a.pg, row, 2 * c, h, there0);
    tile_at<D>(a.pg, row, min(2 * c + 1, n_tiles - 1), h, there1);
    const int lim0 = there0 ? min(ctx - 32 * c, 16) : 0, lim1 = there1 ? min(max(ctx - 32 * c - 16, 0), 16) : 0;
    s[0] *= a.scale_log2e;
    s[1] *= a.scale_log2e;
    // what lies in a masked place may be anything: scores are replaced, and values cleared (0 times infinity is no 0).  Without a
    // branch: one around the fragments sends them through scratch memory.
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[0][r] = 4 * g + r < lim0 ? s[0][r] : -INFINITY;
      s[1][r] = 4 * g + r < lim1 ? s[1][r] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int keep = (i ? lim1 : lim0) - 4 * g;
      const uint32_t lo = keep >= 2 ? ~0u : keep == 1 ? 0xffffu : 0u, hi = keep >= 4 ? ~0u : keep == 3 ? 0xffffu : 0u;
      const u32x4 mask = {lo, hi, lo, hi};
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) x.V[i][kk] &= mask;
    }
    if (n < G) {
      *reinterpret_cast<f32x4*>(score_row + 32 * c + 4 * g) = s[0];
      if (2 * c + 1 < n_tiles) *reinterpret_cast<f32x4*>(score_row + 32 * c + 16 + 4 * g) = s[1];
    }
    float mc = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) mc = fmaxf(mc, fmaxf(s[0][r], s[1][r]));
    mc = xor_max<32>(xor_max<16>(mc));
    const float mn = fmaxf(m, mc), ms = mn == -INFINITY ? 0.f : mn;
    float p[8], ps = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - ms);
      ps += p[i];
    }
    if (__any(mn != m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - ms);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < 2 * DB; ++j) acc[j] *= alpha;
      m = mn;
    }
    l += ps;
    u32x4 ph, pl;  // P to some 16 bits: the product's share of the error stays below the output's rounding
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ph[i] = pack_bf(p[2 * i], p[2 * i + 1]);
      pl[i] = pack_bf(p[2 * i] - lo_bf(ph[i]), p[2 * i + 1] - hi_bf(ph[i]));
    }
    auto half = [](const u32x4& v, int hf) { return __builtin_bit_cast(s16x4, u32x2{v[hf], v[hf + 1]}); };
#pragma unroll
    for (int part = 0; part < 4; ++part) {  // (tile 0, hi), (tile 0, lo), (tile 1, hi), (tile 1, lo)
      const s16x4 pb = half((part & 1) ? pl : ph, (part >> 1) * 2);
#pragma unroll
      for (int j = 0; j < 2 * DB; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(half(x.V[part >> 1][j >> 1], (j & 1) * 2), pb, acc[j], 0, 0, 0);
    }
  };

  Chunk<DB> A, B;
  if (c0 + 1 < c1) {
    int c = c0;
    load(c, A);
    load(c + 1, B);
    for (; c + 3 < c1; c += 2) {  // both buffers have a successor
      attend(c, A);
      load(c + 2, A);
      attend(c + 1, B);
      load(c + 3, B);
    }
    attend(c, A);
    if (c + 2 < c1) {
      load(c + 2, A);
      attend(c + 1, B);
      attend(c + 2, A);
    } else {
      attend(c + 1, B);
    }
  } else if (c0 < c1) {
    load(c0, A);
    attend(c0, A);
  }

  l = xor_sum<32>(xor_sum<16>(l));
  if (n < G) {
#pragma unroll
    for (int j = 0; j < 2 * DB; ++j) *reinterpret_cast<f32x4*>(&sm_o[wave][n][j * 16 + 4 * g]) = acc[j];
    if (g == 0) {
      sm_m[wave][n] = m;
      sm_l[wave][n] = l;
    }
  }
  __threadfence_block();  // the scores, for the last loop
  __syncthreads();
  for (int idx = threadIdx.x; idx < G * D; idx += DW * 64) {
    const int hn = idx / D, d = idx % D;
    float M = sm_m[0][hn];
#pragma unroll
    for (int w = 1; w < DW; ++w) M = fmaxf(M, sm_m[w][hn]);
    const float ms = M == -INFINITY ? 0.f : M;  // every token masked: weights of zero
    float o = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < DW; ++w) {
      const float e = __builtin_amdgcn_exp2f(sm_m[w][hn] - ms);
      o += e * sm_o[w][hn][d];
      L += e * sm_l[w][hn];
    }
    if (a.splits == 1) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      a.out[(row0 + hn) * D + d] = f2bf(o * inv);
      if (d == 0) {
        sm_M[hn] = ms;
        sm_inv[hn] = inv;
      }
    } else {
      const int64_t at = (row0 + hn) * a.splits + split;
      a.part_o[at * D + d] = o;
      if (d == 0) {
        a.part_ml[at * 2] = M;
        a.part_ml[at * 2 + 1] = L;
      }
    }
  }
  if (a.splits > 1) return;
  __syncthreads();
  if (now == nullptr) return;
  const int end = (int)min((int64_t)ctx, a.rows.len);
  for (int j = threadIdx.x; j < end; j += DW * 64) {
    float w = 0.f;
#pragma unroll 4
    for (int hn = 0; hn < G; ++hn) w += __builtin_amdgcn_exp2f(a.scores[(row0 + hn) * a.pg.cap + j] - sm_M[hn]) * sm_inv[hn];
    now[j] = (j < ctx - 1 && had != nullptr ? had[j] : 0.f) + w;
  }
}

// joins the splits: grid (kv heads, shares of the context, batch), 4 waves.  A few dependent reads long, so what does not depend on the sums - the
// scores of a thread's first token, its mass so far - is asked for ahead of them.
template <int D>
__global__ __launch_bounds__(256) void decode_mass_join_kernel(DecodeMass a) {
  __shared__ float sm_M[16], sm_inv[16], sm_e[16][MAX_SPLITS];
  const int h = blockIdx.x, b = blockIdx.z, G = a.G, lane = threadIdx.x & 63;
  const int64_t row0 = (int64_t)b * a.pg.n_kv * G + (int64_t)h * G;
  const int ctx = min(max(a.lens[b], 0), a.pg.cap), end = (int)min((int64_t)ctx, a.rows.len);
  const float* const had = a.rows.in(b, h);
  float* const now = a.rows.out(b, h);
  const float* const scores = a.scores + row0 * a.pg.cap;
  int j = blockIdx.y * 256 + threadIdx.x;
  auto old = [&](int at) { return at < ctx - 1 && had != nullptr ? had[at] : 0.f; };
  const bool first = now != nullptr && j < end;
  float s[16], was = 0.f;
  if (first) {
#pragma unroll
    for (int hn = 0; hn < 16; ++hn)
      if (hn < G) s[hn] = scores[(int64_t)hn * a.pg.cap + j];
    was = old(j);
  }
  for (int hn = threadIdx.x >> 6; hn < G; hn += 4) {
    const bool on = lane < a.splits;
    const float2 ml = on ? *reinterpret_cast<const float2*>(a.part_ml + ((row0 + hn) * a.splits + lane) * 2) : float2{-INFINITY, 0.f};
    const float M = wave_max(ml.x), ms = M == -INFINITY ? 0.f : M;
    const float e = __builtin_amdgcn_exp2f(ml.x - ms), L = wave_sum(e * ml.y);
    sm_e[hn][lane] = e;
    if (lane == 0) {
      sm_M[hn] = ms;
      sm_inv[hn] = L == 0.f ? 0.f : 1.f / L;
    }
  }
  __syncthreads();
  if (first) {
    float w = 0.f;
#pragma unroll
    for (int hn = 0; hn < 16; ++hn)
      if (hn < G) w += __builtin_amdgcn_exp2f(s[hn] - sm_M[hn]) * sm_inv[hn];
    now[j] = was + w;
    for (j += gridDim.y * 256; j < end; j += gridDim.y * 256) {
      w = 0.f;
#pragma unroll 8
      for (int hn = 0; hn < G; ++hn) w += __builtin_amdgcn_exp2f(scores[(int64_t)hn * a.pg.cap + j] - sm_M[hn]) * sm_inv[hn];
      now[j] = old(j) + w;
    }
  }
  for (int idx = blockIdx.y * 256 + threadIdx.x; idx < G * D; idx += gridDim.y * 256) {
    const int hn = idx / D, d = idx % D;
    float o = 0.f;
    for (int p = 0; p < a.splits; p += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = a.part_o[((row0 + hn) * a.splits + min(p + i, a.splits - 1)) * D + d];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = p + i < a.splits ? sm_e[hn][p + i] : 0.f;
        o += e != 0.f ? e * v[i] : 0.f;  // (an empty split wrote no sums)
      }
    }
    a.out[(row0 + hn) * D + d] = f2bf(o * sm_inv[hn]);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// prompt
//
// The rows of a (sequence, kv head) are the G query heads of its observed query tokens, token-major: row r is head r % G of token
// r / G, so that what rows see grows with their number.  Three launches: the rows' maxima and sums (and their q rows in the matrix
// operand's order), the join of those where the keys were split, the column sums of exp2(score - log2 of the row's sum).  Both product
// loops hold one side in registers and stream the other, S^T = K Q^T on 32x32x16: a lane then has one row and 16 keys of it, and
// neither the running maximum and sum nor the column sums leave the lane before the end.
//
// Bound by the matrix cores at the clock that random operands leave them, and the powers beside them (a score: 8 cycles of matrix instruction,
// 16 of fma, exp2 and sum): 240 us each walk for 4096 rows of 32 heads on 8 behind 4096 tokens (206 GFLOP: 860 TFLOP/s), 47 + 47 for the last 64
// rows of 64 heads over 32768; and by launches and dependent reads for short ones, 6 + 7 us for 137 rows.
// ---------------------------------------------------------------------------------------------------------------------
struct PromptMass {
  const uint16_t* q;
  int64_t q_stride;
  const uint16_t* kc;
  Pages pg;
  const int32_t *cu, *kv_lens;
  MassRows rows;
  uint16_t* packed;  // [n_kv][tiles][D * 32] rows in operand order
  float* part_ml;    // [n_kv][parts][tiles * 32][2]
  float* lse;        // [n_kv][tiles * 32]: log2 of the row's sum of exp2, infinity for a row that sees nothing
  int64_t tiles;     // 32-row tiles of a kv head, all sequences
  int n_tokens, window, max_rows, G, parts;
  float scale_log2e;
};

struct PromptSeq {
  int q_begin;     // first observed token's row of q
  int n_rows;      // G * observed tokens
  int kv, fresh;   // cached tokens; the first of them that this step stored
  int first;       // position of the first observed token
  int64_t tile0;   // first 32-row tile
};

__device__ __forceinline__ PromptSeq prompt_seq(const PromptMass& a, int b) {
  PromptSeq s;
  const int begin = min(max(a.cu[b], 0), a.n_tokens), end = min(max(a.cu[b + 1], begin), a.n_tokens);
  const int len = a.kv_lens[b], seen = min(end - begin, a.max_rows);
  s.kv = min(max(len, 0), a.pg.cap);
  s.fresh = max(len, 0) - (end - begin);
  s.q_begin = end - seen;
  s.first = len - seen;
  s.n_rows = seen * a.G;
  s.tile0 = a.window > 0 ? (int64_t)b * ((a.max_rows * a.G + 31) >> 5) : (((int64_t)begin * a.G) >> 5) + b;
  return s;
}

// token of the 32 that register r of lane half `hf` holds
__device__ __forceinline__ int key_of(int r, int hf) { return (r >> 2) * 8 + hf * 4 + (r & 3); }

// ---- the row sums: a wave's 64 rows, two tiles of 32
template <int D>
struct RowTiles {
  static constexpr int J = D / 16;
  u32x4 Q[2][J];
  int limit[2];                      // keys that the lane's row sees
  float m[2], shift[2], l[2];        // reference point, what is added to a score (its negative; infinity before there is one), sum
  int64_t tile;
  bool second;                       // the second tile is there
  int all, most;                     // keys that every row sees, that the last one sees

  // rows group * 64 on, of which there is one at least
  __device__ __forceinline__ void load(const PromptMass& a, const PromptSeq& sq, int h, int group, int lane, bool pack) {
    const int hf = lane >> 5;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = group * 64 + t * 32 + (lane & 31);
      const bool on = r < sq.n_rows;
      const int token = on ? r / a.G : 0;
      limit[t] = on ? min(sq.first + token + 1, sq.kv) : 0;
      const uint16_t* p = a.q + (int64_t)(sq.q_begin + token) * a.q_stride + (int64_t)(h * a.G + (on ? r - token * a.G : 0)) * D + 8 * hf;
#pragma unroll
      for (int j = 0; j < J; ++j) Q[t][j] = on ? *reinterpret_cast<const u32x4*>(p + 16 * j) : u32x4{0, 0, 0, 0};
      m[t] = -INFINITY, shift[t] = INFINITY, l[t] = 0.f;
    }
    tile = sq.tile0 + group * 2;
    second = group * 64 + 32 < sq.n_rows;
    all = group * 64 + 64 <= sq.n_rows ? min(sq.first + group * 64 / a.G + 1, sq.kv) : 0;
    most = max(min(sq.first + min(group * 64 + 63, sq.n_rows - 1) / a.G + 1, sq.kv), 0);
    if (pack) {
      uint16_t* to = a.packed + (h * a.tiles + tile) * (32 * D) + lane * 8;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (t == 0 || second)
#pragma unroll
          for (int j = 0; j < J; ++j) *reinterpret_cast<u32x4*>(to + t * (32 * D) + j * 512) = Q[t][j];
    }
  }
  // The reference point only has to be near the maximum (32 bits hold sums of up to 2^8 as they do those of up to 1), and a sum of 16 powers tells
  // whether it is: no maximum is taken while the sums stay below.  Infinite until a key was seen, so that the first one comes here.
  __device__ __forceinline__ float move_to(int t, float mx) {
    const float mn = fmaxf(m[t], mx), to = mn == -INFINITY ? 0.f : -mn;
    l[t] *= __builtin_amdgcn_exp2f(m[t] + to);
    m[t] = mn;
    shift[t] = mn == -INFINITY ? INFINITY : -mn;
    return to;
  }
  __device__ __forceinline__ void add_plain(int t, const f32x16& s, float now, float scale) {
    if (__any(!(now <= 256.f))) {
      float mx = -INFINITY, part[4] = {};
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r] * scale);
      const float to = move_to(t, mx);
#pragma unroll
      for (int r = 0; r < 16; ++r) part[r & 3] += __builtin_amdgcn_exp2f(fmaf(s[r], scale, to));
      now = (part[0] + part[1]) + (part[2] + part[3]);
    }
    l[t] += now;
  }
  __device__ __forceinline__ void multiply(const u32x4 (&K)[J], f32x16 (&s)[2]) const {
    s[0] = f32x16{};
    s[1] = f32x16{};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(K[j]), as_frag(Q[0][j]), s[0], 0, 0, 0);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(K[j]), as_frag(Q[1][j]), s[1], 0, 0, 0);
    }
  }
  // key tile k, of which rows see a part or whose pages may not be there
  __device__ __forceinline__ void add_masked(const f32x16 (&s)[2], int k, int hf, bool there0, bool there1, float scale) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      // (against constants: sums of the lane's own cost a register each)
      const int mine = limit[t] - 32 * k - 4 * hf, lim0 = there0 ? mine : 0, lim1 = there1 ? mine : 0;
      auto seen = [&](int r) { return key_of(r, 0) < (r < 8 ? lim0 : lim1); };
      float mx = -INFINITY, part[4] = {};
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, seen(r) ? s[t][r] * scale : -INFINITY);
      const float to = move_to(t, mx);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[t][r], scale, to));
        part[r & 3] += seen(r) ? e : 0.f;
      }
      l[t] += (part[0] + part[1]) + (part[2] + part[3]);
    }
  }
  // a row's reference point and sum (both lane halves have part of it)
  __device__ __forceinline__ float2 total(int t) const {
    const float mo = __shfl_xor(m[t], 32, 64), lo = __shfl_xor(l[t], 32, 64);
    const float M = fmaxf(m[t], mo), to = M == -INFINITY ? 0.f : -M;
    return {M, l[t] * __builtin_amdgcn_exp2f(m[t] + to) + lo * __builtin_amdgcn_exp2f(mo + to)};
  }
};
__device__ __forceinline__ void store_row(const PromptMass& a, int h, int part, int64_t at, float2 ml) {
  if (a.parts == 1) a.lse[h * a.tiles * 32 + at] = ml.y == 0.f ? INFINITY : ml.x + __builtin_amdgcn_logf(ml.y);
  else reinterpret_cast<float2*>(a.part_ml)[(h * (int64_t)a.parts + part) * a.tiles * 32 + at] = ml;
}

// A workgroup has 64 rows and its waves every fourth key tile of a part of the keys, whose fragments come straight from the cache, a tile ahead; the
// waves join in LDS.  Three waves share a SIMD's matrix core (two: 699 us against 616 for 8192 rows of 64 heads on 8, 122 against 108 for 4 x 2048 of 32;
// keys by way of LDS, shared by four waves of 64 rows, with the products of a tile written among the powers of the one before: 613 and 113).
// grid (kv heads, row groups x parts of the keys, sequences)
template <int D>
__global__ __launch_bounds__(256, 3) void prompt_rows_kernel(PromptMass a) {
  constexpr int J = D / 16;
  __shared__ float2 sm[4][64];
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5;
  // the rows that see most first
  const int part = blockIdx.y % a.parts, group = ((sq.n_rows + 63) >> 6) - 1 - (int)(blockIdx.y / a.parts);
  if (group < 0) return;  // uniform for the workgroup
  RowTiles<D> x;
  x.load(a, sq, h, group, lane, part == 0 && wave == 0);
  const int tiles = (x.most + 31) >> 5, share = (tiles + a.parts - 1) / a.parts, k1 = min((part + 1) * share, tiles);
  const int32_t* row = a.pg.table + (int64_t)b * a.pg.table_stride;
  const int last_tile = max((sq.kv + 15) / 16 - 1, 0);
  struct Tile {
    u32x4 K[J];
    bool there0, there1;
  };
  auto load = [&](int k, Tile& t) __attribute__((always_inline)) {
    const int64_t at0 = tile_at<D>(a.pg, row, min(2 * k, last_tile), h, t.there0);
    const int64_t at1 = tile_at<D>(a.pg, row, min(2 * k + 1, last_tile), h, t.there1);
    const uint16_t* p = a.kc + ((lane & 16) ? at1 : at0) + (hf * 16 + (lane & 15)) * 8;
#pragma unroll
    for (int j = 0; j < J; ++j) t.K[j] = *reinterpret_cast<const u32x4*>(p + (j >> 1) * 512 + (j & 1) * 256);
  };
  auto add = [&](int k, const Tile& t) __attribute__((always_inline)) {
    f32x16 s[2];
    x.multiply(t.K, s);
    if (t.there0 && t.there1 && 32 * k + 32 <= x.all) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum[4] = {};
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r & 3] += __builtin_amdgcn_exp2f(fmaf(s[i][r], a.scale_log2e, x.shift[i]));
        x.add_plain(i, s[i], (sum[0] + sum[1]) + (sum[2] + sum[3]), a.scale_log2e);
      }
    } else {
      x.add_masked(s, k, hf, t.there0, t.there1, a.scale_log2e);
    }
  };
  int k = part * share + wave;
  if (k < k1) {
    Tile A, B;
    load(k, A);
    while (true) {
      load(min(k + 4, k1 - 1), B);
      add(k, A);
      if ((k += 4) >= k1) break;
      load(min(k + 4, k1 - 1), A);
      add(k, B);
      if ((k += 4) >= k1) break;
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float2 ml = x.total(t);
    if (lane < 32) sm[wave][t * 32 + lane] = ml;
  }
  __syncthreads();
  if (wave != 0 || (lane >= 32 && !x.second)) return;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w][lane].x);
  const float to = M == -INFINITY ? 0.f : -M;
#pragma unroll
  for (int w = 0; w < 4; ++w) L += sm[w][lane].y * __builtin_amdgcn_exp2f(sm[w][lane].x + to);
  store_row(a, h, part, x.tile * 32 + lane, {M, L});
}

__global__ __launch_bounds__(256) void prompt_join_kernel(PromptMass a) {
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int r = blockIdx.y * 256 + threadIdx.x;
  if (r >= ((sq.n_rows + 31) & ~31)) return;
  const int64_t at = sq.tile0 * 32 + r;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + h * (int64_t)a.parts * a.tiles * 32 + at;
  float M = -INFINITY, L = 0.f;
  for (int p = 0; p < a.parts; p += 8) {
    float2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p + i < a.parts ? ml[(p + i) * a.tiles * 32] : float2{-INFINITY, 0.f};
    float mn = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) mn = fmaxf(mn, v[i].x);
    const float to = mn == -INFINITY ? 0.f : -mn;
    L *= __builtin_amdgcn_exp2f(M + to);
#pragma unroll
    for (int i = 0; i < 8; ++i) L += v[i].y * __builtin_amdgcn_exp2f(v[i].x + to);
    M = mn;
  }
  a.lse[h * a.tiles * 32 + at] = L == 0.f ? INFINITY : M + __builtin_amdgcn_logf(L);
}

// ---- the column sums: a wave's 64 keys, two tiles of 32
template <int D>
struct Keys {
  static constexpr int J = D / 16;
  u32x4 K[2][J];
  bool there[4];  // 16-token page tiles
  bool whole;     // all of them, and all tokens in the context
  f32x16 sum[2];
  __device__ __forceinline__ void load(const PromptMass& a, const PromptSeq& sq, int b, int h, int key0, int lane) {
    const int32_t* row = a.pg.table + (int64_t)b * a.pg.table_stride;
    const int last_tile = (sq.kv + 15) / 16 - 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      // 32 keys as the A operand: lane (half, t) has dims 16 j + 8 half .. + 7 of token t
      const int k = key0 / 16 + 2 * t;
      const int64_t at0 = tile_at<D>(a.pg, row, min(k, last_tile), h, there[2 * t]);
      const int64_t at1 = tile_at<D>(a.pg, row, min(k + 1, last_tile), h, there[2 * t + 1]);
      const uint16_t* p = a.kc + ((lane & 16) ? at1 : at0) + ((lane >> 5) * 16 + (lane & 15)) * 8;
#pragma unroll
      for (int j = 0; j < J; ++j) K[t][j] = *reinterpret_cast<const u32x4*>(p + (j >> 1) * 512 + (j & 1) * 256);
      sum[t] = f32x16{};
    }
    whole = there[0] && there[1] && there[2] && there[3] && key0 + 64 <= sq.kv;
  }
  // the first row that sees a key
  static __device__ __forceinline__ int sees(const PromptMass& a, const PromptSeq& sq, int key) {
    return (int)min((int64_t)max(key - sq.first, 0) * a.G, (int64_t)sq.n_rows);
  }
  // row tile i's powers, where some rows do not see all keys or are behind the last
  __device__ __forceinline__ void add_masked(const PromptMass& a, const PromptSeq& sq, int i, const f32x16 (&s)[2], float log_sum, int key0, int lane) {
    const int rr = i * 32 + (lane & 31), limit = rr < sq.n_rows ? min(sq.first + rr / a.G + 1, sq.kv) : 0;
    const int mine = limit - key0 - 4 * (lane >> 5);  // (against constants: sums of the lane's own cost a register each)
    float shift = -log_sum;
    asm volatile("" : "+v"(shift));  // (or what both kinds of powers begin with is taken ahead of the branch between them, into 32 registers)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int lim0 = there[2 * t] ? mine : 0, lim1 = there[2 * t + 1] ? mine : 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale_log2e, shift));
        sum[t][r] += 32 * t + key_of(r, 0) < (r < 8 ? lim0 : lim1) ? p : 0.f;
      }
    }
  }
  // the sums over the lanes' rows to 64 places
  __device__ __forceinline__ void reduce(float* to, int lane) const {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v = xor_sum<1>(sum[t][r]);
        v = xor_sum<2>(v);
        v = xor_sum<4>(v);
        v = xor_sum<8>(v);
        v = xor_sum<16>(v);
        if ((lane & 31) == 0) to[32 * t + key_of(r, lane >> 5)] = v;
      }
  }
};

// A workgroup has KW times 64 keys and 4 / KW waves for each, which take every (4 / KW)-th tile of the rows from the packed copy, a tile ahead; they
// join in LDS.  With 128 dims two waves a SIMD and two sets of row registers (three and one set: 671 us against 615 for 8192 rows of 64 heads on 8).
// grid (kv heads, key blocks, sequences)
template <int D, int KW>
__global__ __launch_bounds__(256, D == 128 ? 2 : 3) void prompt_columns_kernel(PromptMass a) {
  constexpr int J = D / 16, TILE = 32 * D, RW = 4 / KW;
  __shared__ float sm[4][64];
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW;
  const int key0 = ((int)blockIdx.y * KW + wave / RW) * 64, j = key0 + lane;
  if ((int)blockIdx.y * KW * 64 >= sq.kv) return;  // uniform for the workgroup
  Keys<D> x;
  x.load(a, sq, b, h, key0, lane);
  const float *const had = a.rows.in(b, h);
  float* const now = a.rows.out(b, h);
  const bool mine = rw == 0 && j < sq.kv && j < a.rows.len && now != nullptr;  // the key that the lane writes
  const float was = mine && j < sq.fresh && had != nullptr ? had[j] : 0.f;
  // row tiles: from the first that has a row which sees a key; those all of whose rows are there and see all keys
  const int tiles = key0 < sq.kv ? (sq.n_rows + 31) >> 5 : 0;
  const int first = x.sees(a, sq, key0) >> 5, plain_from = x.whole ? (x.sees(a, sq, key0 + 63) + 31) >> 5 : tiles, plain_to = sq.n_rows >> 5;
  const uint16_t* const packed = a.packed + (h * a.tiles + sq.tile0) * TILE + lane * 8;
  const float* const lses = a.lse + (h * a.tiles + sq.tile0) * 32 + (lane & 31);
  struct Rows {
    u32x4 Q[J];
    float lse;
  };
  auto load = [&](int i, Rows& r) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < J; ++j) r.Q[j] = *reinterpret_cast<const u32x4*>(packed + (int64_t)i * TILE + j * 512);
    r.lse = lses[i * 32];
  };
  auto add = [&](int i, const Rows& r) __attribute__((always_inline)) {
    f32x16 s[2] = {{}, {}};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(x.K[0][j]), as_frag(r.Q[j]), s[0], 0, 0, 0);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(x.K[1][j]), as_frag(r.Q[j]), s[1], 0, 0, 0);
    }
    if (i >= plain_from && i < plain_to) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r_ = 0; r_ < 16; ++r_) x.sum[t][r_] += __builtin_amdgcn_exp2f(fmaf(s[t][r_], a.scale_log2e, -r.lse));
    } else {
      x.add_masked(a, sq, i, s, r.lse, key0, lane);
    }
  };
  // From the last rows, which all keys see, to the first: workgroups that start together read the same rows at the same time, from their
  // XCD's L2.
  int i = tiles - 1 - rw;
  if (i >= first) {
    Rows A, B;
    load(i, A);
    while (true) {
      load(max(i - RW, first), B);
      add(i, A);
      if ((i -= RW) < first) break;
      load(max(i - RW, first), A);
      add(i, B);
      if ((i -= RW) < first) break;
    }
  }
  x.reduce(sm[wave], lane);
  __syncthreads();
  if (!mine) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < RW; ++w) v += sm[wave + w][lane];
  now[j] = was + v;
}

struct PromptPlan {
  int max_rows, parts, groups, key_waves;
  int64_t tiles;
  size_t packed, lse, ml;  // bytes
  size_t bytes() const { return packed + lse + ml; }
};

PromptPlan prompt_plan(int n_seqs, int64_t n_tokens, int max_seqlen_q, int window, int n_q, int n_kv, int D, int64_t cap) {
  PromptPlan p;
  const int G = n_q / n_kv;
  p.max_rows = window > 0 ? std::min(window, max_seqlen_q) : max_seqlen_q;
  p.tiles = window > 0 ? (int64_t)n_seqs * (((int64_t)p.max_rows * G + 31) / 32) : n_tokens * G / 32 + n_seqs;
  p.groups = (int)(((int64_t)p.max_rows * G + 63) / 64);
  const int64_t units = std::max<int64_t>((int64_t)n_seqs * n_kv, 1), blocks = units * p.groups, key_blocks = units * ((cap + 255) / 256);
  // parts of the keys until there are two workgroups a CU, of 512 keys at least: below that their join costs more
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + blocks - 1) / blocks, cap / 512, 64}));
  // four waves for 64 keys, so that the rows are split as well - except for so many keys that they fill the chip and rows so few (below 2048 of a kv
  // head) that a wave's keys take longer to come than the rows: 64 rows of 64 heads on 8 over 32768 keys, 49 us against 62
  p.key_waves = key_blocks >= 256 && p.groups < 32 ? 4 : 1;
  p.packed = (size_t)n_kv * p.tiles * 32 * D * 2;
  p.lse = (size_t)n_kv * p.tiles * 32 * 4;
  p.ml = p.parts > 1 ? (size_t)n_kv * p.tiles * 32 * 8 * p.parts : 0;
  return p;
}

template <int D>
void launch_prompt(const PromptMass& a, const PromptPlan& p, int n_kv, int n_seqs, int64_t cap, hipStream_t stream) {
  prompt_rows_kernel<D><<<dim3(n_kv, (unsigned)(p.groups * p.parts), n_seqs), 256, 0, stream>>>(a);
  if (p.parts > 1) prompt_join_kernel<<<dim3(n_kv, (p.groups * 64 + 255) / 256, n_seqs), 256, 0, stream>>>(a);
  if (p.key_waves == 4) prompt_columns_kernel<D, 4><<<dim3(n_kv, (unsigned)((cap + 255) / 256), n_seqs), 256, 0, stream>>>(a);
  else prompt_columns_kernel<D, 1><<<dim3(n_kv, (unsigned)((cap + 63) / 64), n_seqs), 256, 0, stream>>>(a);
}

// A workgroup fills a CU (with 64-wide heads half of one).  256 units and more are left whole, whatever the lengths of their contexts (32 sequences of
// 1024 tokens on 8 kv heads, 128-wide: 25 us, in two halves each 26 + 4; 64-wide, 32 heads: 14 us, 73 MB at 5.3 TB/s); fewer are split into some
// four workgroups a CU, so that contexts of all lengths share the chip evenly (24 sequences of 101 to 8000 tokens on 4
// kv heads: 55 us with one a CU, 48 with four), of 256 tokens at least.
int decode_splits(int batch, int n_kv, int64_t cap) {
  const int64_t units = std::max<int64_t>((int64_t)batch * n_kv, 1);
  if (units >= 256) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({1024 / units, (cap + 32 * DW - 1) / (32 * DW), MAX_SPLITS}));
}

size_t decode_bytes(int batch, int n_q, int D, int splits, int64_t cap) {
  const size_t rows = (size_t)batch * n_q;
  return rows * cap * 4 + (splits > 1 ? rows * splits * (D + 2) * 4 : 0);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" size_t mi_paged_attn_decode_mass_workspace(int batch, int n_q_heads, int n_kv_heads, int head_dim, int block_size, int table_width) {
  if (batch <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || block_size <= 0 || table_width <= 0) return 0;
  const int64_t cap = (int64_t)block_size * table_width;
  return decode_bytes(batch, n_q_heads, head_dim, decode_splits(batch, n_kv_heads, cap), cap);
}

extern "C" int mi_paged_attn_decode_mass(const mi_bf16* q, int64_t q_row_stride, const mi_bf16* k_cache, const mi_bf16* v_cache,
                                         int64_t num_blocks, const int32_t* block_table, int64_t table_stride, int table_width,
                                         const int32_t* context_lens, float* mass, int64_t mass_rows, int64_t mass_len,
                                         const int32_t* slots, const int32_t* slots_out, mi_bf16* out, void* workspace, size_t ws_bytes,
                                         int batch, int n_q_heads, int n_kv_heads, int head_dim, int block_size, float scale,
                                         mi_stream stream) {
  if (batch < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || num_blocks <= 0 || table_width <= 0 ||
      table_stride < table_width || mass_rows < 0 || mass_len < 0 || block_size <= 0)
    return MI_EINVAL;
  const int64_t cap = (int64_t)block_size * table_width;
  if ((head_dim != 64 && head_dim != 128) || n_q_heads / n_kv_heads > 16 || block_size % 16 != 0 || cap >= (1 << 30) || batch > 65535 ||
      n_kv_heads > 65535)
    return MI_EUNSUPPORTED;
  if (batch == 0) return MI_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_table == nullptr || context_lens == nullptr || mass == nullptr ||
      slots == nullptr || slots_out == nullptr || out == nullptr || workspace == nullptr)
    return MI_EINVAL;
  if (!aligned16(q) || q_row_stride % 8 != 0 || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(workspace))
    return MI_EINVAL;
  const int splits = decode_splits(batch, n_kv_heads, cap);
  if (ws_bytes < decode_bytes(batch, n_q_heads, head_dim, splits, cap)) return MI_EWORKSPACE;
  const size_t rows = (size_t)batch * n_q_heads;
  DecodeMass a;
  a.q = q, a.q_stride = q_row_stride, a.kc = k_cache, a.vc = v_cache;
  a.pg = {block_table, table_stride, num_blocks, block_size / 16, tile_shift(block_size), (int)cap, n_kv_heads};
  a.lens = context_lens;
  a.rows = {mass, mass_rows, mass_len, slots, slots_out, n_kv_heads};
  a.out = out;
  a.scores = static_cast<float*>(workspace);
  a.part_o = a.scores + rows * cap;
  a.part_ml = a.part_o + rows * splits * head_dim;
  a.G = n_q_heads / n_kv_heads, a.splits = splits, a.scale_log2e = scale * 1.44269504088896340736f;
  const dim3 grid(n_kv_heads, splits, batch);
  if (head_dim == 128) decode_mass_kernel<4><<<grid, DW * 64, 0, S(stream)>>>(a);
  else decode_mass_kernel<2><<<grid, DW * 64, 0, S(stream)>>>(a);
  if (splits > 1) {
    const int shares = (int)std::max<int64_t>(1, std::min<int64_t>((cap + 255) / 256, 8192 / ((int64_t)batch * n_kv_heads)));
    const dim3 jg(n_kv_heads, shares, batch);
    if (head_dim == 128) decode_mass_join_kernel<128><<<jg, 256, 0, S(stream)>>>(a);
    else decode_mass_join_kernel<64><<<jg, 256, 0, S(stream)>>>(a);
  }
  return check_launch();
}

extern "C" size_t mi_prompt_attn_mass_workspace(int n_seqs, int64_t n_tokens, int max_seqlen_q, int window, int n_q_heads, int n_kv_heads,
                                                int head_dim, int block_size, int table_width) {
  if (n_seqs <= 0 || n_tokens < 0 || max_seqlen_q < 0 || n_kv_heads <= 0 || n_q_heads <= 0 || block_size <= 0 || table_width <= 0) return 0;
  const PromptPlan p =
      prompt_plan(n_seqs, n_tokens, std::max(max_seqlen_q, 1), window, n_q_heads, n_kv_heads, head_dim, (int64_t)block_size * table_width);
  return p.bytes();
}

extern "C" int mi_prompt_attn_mass(const mi_bf16* q, int64_t q_row_stride, int64_t n_tokens, const mi_bf16* k_cache, int64_t num_blocks,
                                   const int32_t* block_table, int64_t table_stride, int table_width, const int32_t* cu_seqlens_q,
                                   const int32_t* kv_lens, int n_seqs, int max_seqlen_q, int window, float* mass, int64_t mass_rows,
                                   int64_t mass_len, const int32_t* slots, const int32_t* slots_out, void* workspace, size_t ws_bytes,
                                   int n_q_heads, int n_kv_heads, int head_dim, int block_size, float scale, mi_stream stream) {
  if (n_seqs < 0 || n_tokens < 0 || max_seqlen_q < 0 || window < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || num_blocks <= 0 ||
      table_width <= 0 || table_stride < table_width || mass_rows < 0 || mass_len < 0 || block_size <= 0)
    return MI_EINVAL;
  const int64_t cap = (int64_t)block_size * table_width;
  const int G = n_q_heads / n_kv_heads;
  if ((head_dim != 64 && head_dim != 128) || G > 16 || block_size % 16 != 0 || cap >= (1 << 30) || n_seqs > 65535 || n_kv_heads > 65535 ||
      n_tokens * G >= (1 << 30) || (int64_t)max_seqlen_q * G >= (1 << 30))
    return MI_EUNSUPPORTED;
  if (n_seqs == 0) return MI_OK;
  if (q == nullptr || k_cache == nullptr || block_table == nullptr || cu_seqlens_q == nullptr || kv_lens == nullptr || mass == nullptr ||
      slots == nullptr || slots_out == nullptr || workspace == nullptr)
    return MI_EINVAL;
  if (!aligned16(q) || q_row_stride % 8 != 0 || !aligned16(k_cache) || !aligned16(workspace)) return MI_EINVAL;
  const PromptPlan p = prompt_plan(n_seqs, n_tokens, std::max(max_seqlen_q, 1), window, n_q_heads, n_kv_heads, head_dim, cap);
  if (ws_bytes < p.bytes()) return MI_EWORKSPACE;
  if ((int64_t)p.groups * p.parts > 65535 || (cap + 63) / 64 > 65535) return MI_EUNSUPPORTED;
  PromptMass a;
  a.q = q, a.q_stride = q_row_stride, a.kc = k_cache;
  a.pg = {block_table, table_stride, num_blocks, block_size / 16, tile_shift(block_size), (int)cap, n_kv_heads};
  a.cu = cu_seqlens_q, a.kv_lens = kv_lens;
  a.rows = {mass, mass_rows, mass_len, slots, slots_out, n_kv_heads};
  char* ws = static_cast<char*>(workspace);
  a.packed = reinterpret_cast<uint16_t*>(ws);
  a.lse = reinterpret_cast<float*>(ws + p.packed);
  a.part_ml = reinterpret_cast<float*>(ws + p.packed + p.lse);
  a.tiles = p.tiles;
  a.n_tokens = (int)n_tokens, a.window = window, a.max_rows = std::min(p.max_rows, max_seqlen_q), a.G = G, a.parts = p.parts;
  a.scale_log2e = scale * 1.44269504088896340736f;
  if (head_dim == 128) launch_prompt<128>(a, p, n_kv_heads, n_seqs, cap, S(stream));
  else launch_prompt<64>(a, p, n_kv_heads, n_seqs, cap, S(stream));
  return check_launch();
}
