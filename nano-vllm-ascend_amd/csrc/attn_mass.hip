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
  int cap;        // tokens that a table row has room for
  int n_kv;
};

// element offset of tile t of (table row, kv head); `there`: the row names a block of the cache (reads go to block 0 otherwise)
template <int D>
__device__ __forceinline__ int64_t tile_at(const Pages& pg, const int32_t* row, int t, int h, bool& there) {
  const int bi = t / pg.tpb;
  const int32_t blk = row[bi];
  there = blk >= 0 && blk < pg.num_blocks;
  return (((there ? (int64_t)blk : 0) * pg.n_kv + h) * pg.tpb + (t - bi * pg.tpb)) * (16 * D);
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
    mc = fmaxf(mc, __shfl_xor(mc, 16, 64));
    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
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

  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
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
  const float* had = a.rows.in(b, h);
  float* now = a.rows.out(b, h);
  if (now == nullptr) return;
  const int end = (int)min((int64_t)ctx, a.rows.len);
  for (int j = threadIdx.x; j < end; j += DW * 64) {
    float w = 0.f;
    for (int hn = 0; hn < G; ++hn) w += __builtin_amdgcn_exp2f(a.scores[(row0 + hn) * a.pg.cap + j] - sm_M[hn]) * sm_inv[hn];
    now[j] = (j < ctx - 1 && had != nullptr ? had[j] : 0.f) + w;
  }
}

// joins the splits: grid (kv heads, shares of the context, batch), 4 waves
template <int D>
__global__ __launch_bounds__(256) void decode_mass_join_kernel(DecodeMass a) {
  __shared__ float sm_M[16], sm_inv[16], sm_e[16][MAX_SPLITS];
  const int h = blockIdx.x, b = blockIdx.z, G = a.G;
  const int ctx = min(max(a.lens[b], 0), a.pg.cap);
  const int64_t row0 = (int64_t)b * a.pg.n_kv * G + (int64_t)h * G;
  const int lane = threadIdx.x & 63;
  for (int hn = threadIdx.x >> 6; hn < G; hn += 4) {
    const bool on = lane < a.splits;
    const float* ml = a.part_ml + ((row0 + hn) * a.splits + (on ? lane : 0)) * 2;
    const float m = on ? ml[0] : -INFINITY, l = on ? ml[1] : 0.f;
    const float M = wave_max(m), ms = M == -INFINITY ? 0.f : M;
    const float e = __builtin_amdgcn_exp2f(m - ms), L = wave_sum(e * l);
    sm_e[hn][lane] = e;
    if (lane == 0) {
      sm_M[hn] = ms;
      sm_inv[hn] = L == 0.f ? 0.f : 1.f / L;
    }
  }
  __syncthreads();
  for (int idx = blockIdx.y * 256 + threadIdx.x; idx < G * D; idx += gridDim.y * 256) {
    const int hn = idx / D, d = idx % D;
    float o = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float e = sm_e[hn][s];
      if (e != 0.f) o += e * a.part_o[((row0 + hn) * a.splits + s) * D + d];  // (an empty split wrote no sums)
    }
    a.out[(row0 + hn) * D + d] = f2bf(o * sm_inv[hn]);
  }
  const float* had = a.rows.in(b, h);
  float* now = a.rows.out(b, h);
  if (now == nullptr) return;
  const int end = (int)min((int64_t)ctx, a.rows.len);
  for (int j = blockIdx.y * 256 + threadIdx.x; j < end; j += gridDim.y * 256) {
    float w = 0.f;
    for (int hn = 0; hn < G; ++hn) w += __builtin_amdgcn_exp2f(a.scores[(row0 + hn) * a.pg.cap + j] - sm_M[hn]) * sm_inv[hn];
    now[j] = (j < ctx - 1 && had != nullptr ? had[j] : 0.f) + w;
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
  int n_tokens, window, max_rows, G, parts, row_waves;
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

// two page tiles of K as the A operand of 32x32x16: lane (half, t) has dims 16 j + 8 half .. + 7 of token t
template <int D>
__device__ __forceinline__ void load_keys(const uint16_t* kc, int64_t at0, int64_t at1, int lane, u32x4 (&K)[D / 16]) {
  const uint16_t* p = kc + ((lane & 16) ? at1 : at0) + ((lane >> 5) * 16 + (lane & 15)) * 8;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) K[j] = *reinterpret_cast<const u32x4*>(p + (j >> 1) * 512 + (j & 1) * 256);
}

// token of the 32 that register r of lane half `hf` holds
__device__ __forceinline__ int key_of(int r, int hf) { return (r >> 2) * 8 + hf * 4 + (r & 3); }

template <int D>
__device__ __forceinline__ f32x16 products(const u32x4 (&K)[D / 16], const u32x4 (&Q)[D / 16]) {
  f32x16 s = {};
#pragma unroll
  for (int j = 0; j < D / 16; ++j) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(K[j]), as_frag(Q[j]), s, 0, 0, 0);
  return s;
}

// A wave: 64 rows, one part of the keys they see.  grid (kv heads, row blocks x key blocks, sequences)
template <int D>
__global__ __launch_bounds__(256, 2) void prompt_rows_kernel(PromptMass a) {
  constexpr int J = D / 16;
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5;
  const int key_blocks = a.parts / (4 / a.row_waves);
  const int part = (blockIdx.y % key_blocks) * (4 / a.row_waves) + wave / a.row_waves;
  const int groups = (sq.n_rows + 63) >> 6;
  // the rows that see most first
  const int group = groups - 1 - ((blockIdx.y / key_blocks) * a.row_waves + wave % a.row_waves);
  if (group < 0) return;

  u32x4 Q[2][J];
  int limit[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = group * 64 + t * 32 + (lane & 31);
    const bool on = r < sq.n_rows;
    const int token = r / a.G;
    limit[t] = on ? min(sq.first + token + 1, sq.kv) : 0;
    const uint16_t* p = a.q + (int64_t)(sq.q_begin + token) * a.q_stride + (int64_t)(h * a.G + r - token * a.G) * D + 8 * hf;
#pragma unroll
    for (int j = 0; j < J; ++j) Q[t][j] = on ? *reinterpret_cast<const u32x4*>(p + 16 * j) : u32x4{0, 0, 0, 0};
  }
  const int64_t tile = sq.tile0 + group * 2;
  const bool second = group * 64 + 32 < sq.n_rows;  // the group's second tile is there
  if (part == 0) {
    uint16_t* to = a.packed + (h * a.tiles + tile) * (32 * D) + lane * 8;
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (t == 0 || second)
#pragma unroll
        for (int j = 0; j < J; ++j) *reinterpret_cast<u32x4*>(to + t * (32 * D) + j * 512) = Q[t][j];
  }
  // what every row sees, what the last one does
  const int all = min(sq.first + group * 64 / a.G + 1, sq.kv);
  const int most = min(sq.first + min(group * 64 + 63, sq.n_rows - 1) / a.G + 1, sq.kv);
  const bool full = group * 64 + 64 <= sq.n_rows;
  const int steps = (max(most, 0) + 31) >> 5, share = (steps + a.parts - 1) / a.parts;
  const int k0 = min(part * share, steps), k1 = min(k0 + share, steps);
  const int last_tile = max((sq.kv + 15) / 16 - 1, 0);
  const int32_t* row = a.pg.table + (int64_t)b * a.pg.table_stride;

  float m[2] = {-INFINITY, -INFINITY}, shift[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
  u32x4 K[J];
  bool there0, there1;
  auto load = [&](int k) __attribute__((always_inline)) {
    const int64_t at0 = tile_at<D>(a.pg, row, min(2 * k, last_tile), h, there0), at1 = tile_at<D>(a.pg, row, min(2 * k + 1, last_tile), h, there1);
    load_keys<D>(a.kc, at0, at1, lane, K);
  };
  for (int k = k0; k < k1; ++k) {
    load(k);
    const bool plain = there0 && there1 && full && 32 * k + 32 <= all;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 s = products<D>(K, Q[t]);
      s *= a.scale_log2e;
      if (!plain) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * k + key_of(r, hf) >= limit[t] || !(r < 8 ? there0 : there1)) s[r] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
      // the reference point only has to be near the maximum: sums of exp2 up to 2^8 keep their bits as those up to 1 do
      if (__any(mx > m[t] + 8.f)) {
        const float mn = fmaxf(m[t], mx), to = mn == -INFINITY ? 0.f : -mn;
        l[t] *= __builtin_amdgcn_exp2f(m[t] + to);
        m[t] = mn;
        shift[t] = to;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) l[t] += __builtin_amdgcn_exp2f(s[r] + shift[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float mo = __shfl_xor(m[t], 32, 64), lo = __shfl_xor(l[t], 32, 64);
    const float M = fmaxf(m[t], mo), to = M == -INFINITY ? 0.f : -M;
    const float L = l[t] * __builtin_amdgcn_exp2f(m[t] + to) + lo * __builtin_amdgcn_exp2f(mo + to);
    const int64_t at = (tile + t) * 32 + (lane & 31);
    if (hf == 0 && (t == 0 || second)) {
      if (a.parts == 1) {
        a.lse[h * a.tiles * 32 + at] = L == 0.f ? INFINITY : M + __builtin_amdgcn_logf(L);
      } else {
        float* ml = a.part_ml + ((h * (int64_t)a.parts + part) * a.tiles * 32 + at) * 2;
        ml[0] = M;
        ml[1] = L;
      }
    }
  }
}

__global__ __launch_bounds__(256) void prompt_join_kernel(PromptMass a) {
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int r = blockIdx.y * 256 + threadIdx.x;
  if (r >= ((sq.n_rows + 31) & ~31)) return;
  const int64_t at = sq.tile0 * 32 + r;
  float M = -INFINITY, L = 0.f;
  for (int p = 0; p < a.parts; ++p) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + ((h * (int64_t)a.parts + p) * a.tiles * 32 + at) * 2);
    const float mn = fmaxf(M, ml.x), to = mn == -INFINITY ? 0.f : -mn;
    L = L * __builtin_amdgcn_exp2f(M + to) + ml.y * __builtin_amdgcn_exp2f(ml.x + to);
    M = mn;
  }
  a.lse[h * a.tiles * 32 + at] = L == 0.f ? INFINITY : M + __builtin_amdgcn_logf(L);
}

// A wave: 64 keys, all rows that see one of them.  grid (kv heads, blocks of 256 keys, sequences)
template <int D>
__global__ __launch_bounds__(256, 2) void prompt_columns_kernel(PromptMass a) {
  constexpr int J = D / 16;
  __shared__ float sm[4][64];
  const int h = blockIdx.x, b = blockIdx.z;
  const PromptSeq sq = prompt_seq(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5;
  const int key0 = (blockIdx.y * 4 + wave) * 64;
  if (key0 >= sq.kv) return;
  const int32_t* row = a.pg.table + (int64_t)b * a.pg.table_stride;
  const int last_tile = (sq.kv + 15) / 16 - 1;
  u32x4 K[2][J];
  bool there[4];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int k = key0 / 16 + 2 * t;
    const int64_t at0 = tile_at<D>(a.pg, row, min(k, last_tile), h, there[2 * t]);
    const int64_t at1 = tile_at<D>(a.pg, row, min(k + 1, last_tile), h, there[2 * t + 1]);
    load_keys<D>(a.kc, at0, at1, lane, K[t]);
  }
  const bool whole = there[0] && there[1] && there[2] && there[3];
  f32x16 sum[2] = {{}, {}};
  // the first row that sees key0
  const int tiles = (sq.n_rows + 31) >> 5, from = max(key0 - sq.first, 0) * a.G >> 5;
  for (int i = from; i < tiles; ++i) {
    const uint16_t* p = a.packed + (h * a.tiles + sq.tile0 + i) * (32 * D) + lane * 8;
    u32x4 Q[J];
#pragma unroll
    for (int j = 0; j < J; ++j) Q[j] = *reinterpret_cast<const u32x4*>(p + j * 512);
    const float lse = a.lse[h * a.tiles * 32 + (sq.tile0 + i) * 32 + (lane & 31)];
    const int limit = min(sq.first + (i * 32 + (lane & 31)) / a.G + 1, sq.kv);
    const bool plain = whole && key0 + 64 <= min(sq.first + i * 32 / a.G + 1, sq.kv);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f32x16 s = products<D>(K[t], Q);
      if (plain) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[t][r] += __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2e, -lse));
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2e, -lse));
          sum[t][r] += key0 + 32 * t + key_of(r, hf) < limit && there[2 * t + (r >> 3)] ? p : 0.f;
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v = xor_sum<1>(sum[t][r]);
      v = xor_sum<2>(v);
      v = xor_sum<4>(v);
      v = xor_sum<8>(v);
      v = xor_sum<16>(v);
      if ((lane & 31) == 0) sm[wave][32 * t + key_of(r, hf)] = v;
    }
  __threadfence_block();  // (the wave's own part of the array)
  const float* had = a.rows.in(b, h);
  float* now = a.rows.out(b, h);
  const int j = key0 + lane;
  if (now == nullptr || j >= sq.kv || j >= a.rows.len) return;
  now[j] = (j < sq.fresh && had != nullptr ? had[j] : 0.f) + sm[wave][lane];
}

struct PromptPlan {
  int max_rows, row_waves, parts, groups;
  int64_t tiles;
  size_t packed, lse, ml;  // bytes
};

PromptPlan prompt_plan(int n_seqs, int64_t n_tokens, int max_seqlen_q, int window, int n_q, int n_kv, int D, int64_t cap) {
  PromptPlan p;
  const int G = n_q / n_kv;
  p.max_rows = window > 0 ? std::min(window, max_seqlen_q) : max_seqlen_q;
  p.tiles = window > 0 ? (int64_t)n_seqs * (((int64_t)p.max_rows * G + 31) / 32) : n_tokens * G / 32 + n_seqs;
  p.groups = (int)(((int64_t)p.max_rows * G + 63) / 64);
  p.row_waves = p.groups >= 4 ? 4 : p.groups >= 2 ? 2 : 1;
  const int key_waves = 4 / p.row_waves;
  // parts of the keys until every SIMD has two waves, of 128 keys at least
  const int64_t waves = (int64_t)n_seqs * n_kv * p.groups, want = (2048 + waves - 1) / std::max<int64_t>(waves, 1);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({want, (cap + 127) / 128, 64}));
  p.parts = (int)((parts + key_waves - 1) / key_waves * key_waves);
  p.packed = (size_t)n_kv * p.tiles * 32 * D * 2;
  p.lse = (size_t)n_kv * p.tiles * 32 * 4;
  p.ml = p.parts > 1 ? (size_t)n_kv * p.tiles * 32 * 8 * p.parts : 0;
  return p;
}

int decode_splits(int batch, int n_kv, int64_t cap) {
  const int64_t units = (int64_t)batch * n_kv;
  const int64_t by_chip = 256 / std::max<int64_t>(units, 1), by_length = (cap + 32 * DW - 1) / (32 * DW);
  return (int)std::max<int64_t>(1, std::min<int64_t>({by_chip, by_length, MAX_SPLITS}));
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
  a.pg = {block_table, table_stride, num_blocks, block_size / 16, (int)cap, n_kv_heads};
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
    const int shares = (int)std::max<int64_t>(1, std::min<int64_t>((cap + 1023) / 1024, 2048 / ((int64_t)batch * n_kv_heads)));
    const dim3 jg(n_kv_heads, shares, batch);
    if (head_dim == 128) decode_mass_join_kernel<128><<<jg, 256, 0, S(stream)>>>(a);
    else decode_mass_join_kernel<64><<<jg, 256, 0, S(stream)>>>(a);
  }
  return check_launch();
}

extern "C" size_t mi_prompt_attn_mass_workspace(int n_seqs, int64_t n_tokens, int max_seqlen_q, int window, int n_q_heads, int n_kv_heads,
                                                int head_dim, int block_size, int table_width) {
  if (n_seqs <= 0 || n_tokens < 0 || max_seqlen_q <= 0 || n_kv_heads <= 0 || n_q_heads <= 0 || block_size <= 0 || table_width <= 0) return 0;
  const PromptPlan p =
      prompt_plan(n_seqs, n_tokens, max_seqlen_q, window, n_q_heads, n_kv_heads, head_dim, (int64_t)block_size * table_width);
  return p.packed + p.lse + p.ml;
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
  if (ws_bytes < p.packed + p.lse + p.ml) return MI_EWORKSPACE;
  const int64_t row_blocks = (p.groups + p.row_waves - 1) / p.row_waves, key_blocks = p.parts / (4 / p.row_waves);
  if (row_blocks * key_blocks > 65535 || (cap + 255) / 256 > 65535) return MI_EUNSUPPORTED;
  PromptMass a;
  a.q = q, a.q_stride = q_row_stride, a.kc = k_cache;
  a.pg = {block_table, table_stride, num_blocks, block_size / 16, (int)cap, n_kv_heads};
  a.cu = cu_seqlens_q, a.kv_lens = kv_lens;
  a.rows = {mass, mass_rows, mass_len, slots, slots_out, n_kv_heads};
  char* ws = static_cast<char*>(workspace);
  a.packed = reinterpret_cast<uint16_t*>(ws);
  a.lse = reinterpret_cast<float*>(ws + p.packed);
  a.part_ml = reinterpret_cast<float*>(ws + p.packed + p.lse);
  a.tiles = p.tiles;
  a.n_tokens = (int)n_tokens, a.window = window, a.max_rows = std::min(p.max_rows, max_seqlen_q), a.G = G, a.parts = p.parts, a.row_waves = p.row_waves;
  a.scale_log2e = scale * 1.44269504088896340736f;
  const dim3 rg(n_kv_heads, (unsigned)(row_blocks * key_blocks), n_seqs), cg(n_kv_heads, (unsigned)((cap + 255) / 256), n_seqs);
  if (head_dim == 128) prompt_rows_kernel<128><<<rg, 256, 0, S(stream)>>>(a);
  else prompt_rows_kernel<64><<<rg, 256, 0, S(stream)>>>(a);
  if (p.parts > 1) prompt_join_kernel<<<dim3(n_kv_heads, (p.groups * 64 + 255) / 256, n_seqs), 256, 0, S(stream)>>>(a);
  if (head_dim == 128) prompt_columns_kernel<128><<<cg, 256, 0, S(stream)>>>(a);
  else prompt_columns_kernel<64><<<cg, 256, 0, S(stream)>>>(a);
  return check_launch();
}
