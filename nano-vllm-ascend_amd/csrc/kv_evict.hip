// Eviction from the paged cache by attention mass (attn_mass.hip): of a context of more than `keep` tokens each kv head keeps its
// first ones, its newest ones and, of the others, those of the largest mass.
//
//   key_j = (token j is among the first `sinks` or the last `recent` of the sequence, mass_j); kept: the `keep` largest, the lower slot
//   among equals
//
// Kept tokens below `keep` stay where they are; the n-th kept token from behind it goes to the n-th place that becomes free below it.
// Attention does not care in which order a context's slots are, so this is a copy of the movers alone; and as they come from slots at or
// behind `keep` and go to slots below it, no copy reads what another writes: in place, in any order.  What the order loses, a token's
// position in its sequence, is written down per slot (origin) - for slots below evicted[row][0]; tokens that came later are at slot +
// evicted[row][1].
#include <algorithm>

#include "mi_common.hpp"

namespace mi {
namespace {

struct Evict {
  uint16_t *kc, *vc;
  int64_t num_blocks;
  const int32_t *table, *table_out;
  int64_t table_stride, table_out_stride;
  int tpb, cap, n_kv;
  const int32_t* lens;
  int32_t* lens_out;
  float* mass;
  int32_t *origin, *evicted;
  int64_t rows, len;
  const int32_t *slots, *slots_out;
  int keep, sinks, recent;
  int32_t* head;                // [batch][n_kv][2]: what the second launch does, tokens
  int32_t *src, *free, *moved;  // [batch][n_kv][keep]: where each place's token was; places that became free, slots that move there
};

enum { NOTHING = -1, SAME_PLACES = 0, LISTED = 1 };

// order of the masses as unsigned numbers: NaN below -infinity, both zeros alike; ~0u, which no float maps to, for protected tokens
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f);
  if (f != f) return 0u;
  if (f == 0.f) return 0x80000000u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

struct Tokens {
  const float* mass;
  const int32_t* origin;
  int kept, dropped, ctx, sinks, recent;
  __device__ int position(int j) const { return j < kept ? origin[j] : j + dropped; }
  __device__ uint32_t key_at(int position, float m) const { return position < sinks || position >= ctx + dropped - recent ? ~0u : key_of(m); }
  __device__ uint32_t key(int j) const { return key_at(position(j), mass[j]); }
};

// One workgroup per (kv head, sequence): the keep-th largest key digit by digit (11, 11 and 10 bits, counts in LDS), then the lists in slot
// order.  A wave has a contiguous part of the slots, 64 at a time, so that ranks need the waves' totals and ballots only.  Up to HELD tokens the
// keys are kept in LDS; longer contexts are read again in each of the six walks.  Masses share their leading bits, and lanes that add to one address
// wait for one another: two copies of the counts.  10 us for 1100 tokens, 14 for 32 sequences of some 4200, 37 for 8 of 32768 (8 kv heads): barriers
// and dependent reads, then the walks over the keys on one CU.
// (Masses that change between two walks - a call that names a row twice, another stream - make the lists disagree with their counts.  What stays
// is then anyone's guess, but every index taken from a list is held to its range.)
constexpr int CT = 1024, CW = CT / 64, BINS = 2048, COPIES = 2;

struct Counts {
  uint32_t count[BINS * COPIES];
  uint32_t found[3];
  int in_wave[CW], equal[CW], n_free[CW], n_moved[CW];
};

// the sum over lanes 0 .. the lane's own, on the VALU's lane shifts (within 16 lanes, then the last of 16 and of 32 to those behind)
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
// of the waves' numbers in LDS: the sum before this wave's, and of all
__device__ __forceinline__ int before_wave(const int* of_wave, int wave, int lane, int& all) {
  const int s = wave_scan(lane < CW ? of_wave[lane] : 0);
  all = __builtin_amdgcn_readlane(s, CW - 1);
  return wave > 0 ? __builtin_amdgcn_readlane(s, wave - 1) : 0;
}

template <bool IN_LDS>
__device__ __forceinline__ void choose(const Evict& a, const Tokens& tk, Counts& sm, uint32_t* held, float* mass_out, int32_t* origin_out, bool same_row,
                                       int64_t unit) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = ((tk.ctx + CT - 1) / CT) * 64, j0 = min(wave * part, tk.ctx), j1 = min(j0 + part, tk.ctx);
  auto key = [&](int j) { return IN_LDS ? held[j] : tk.key(j); };
  // f(slot, key, the slot is there) for slots from .. to - 1, 64 at a time; four keys are on their way at a time
  auto walk = [&](int from, int to, auto&& f) __attribute__((always_inline)) {
    for (int j = from + lane; j - lane < to; j += 256) {
      uint32_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = j + 64 * i < to ? key(j + 64 * i) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j - lane + 64 * i < to) f(j + 64 * i, k[i], j + 64 * i < to);
    }
  };
  if (IN_LDS) {
    for (int j = tid; j < tk.ctx; j += 8 * CT) {
      float m[8];
      int p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = min(j + CT * i, tk.ctx - 1);
        m[i] = tk.mass[at];
        p[i] = j - tid + CT * i < tk.kept ? tk.origin[min(at, tk.kept - 1)] : 0;  // (the same answer for the whole workgroup)
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = j + CT * i;
        if (at < tk.ctx) held[at] = tk.key_at(at < tk.kept ? p[i] : at + tk.dropped, m[i]);
      }
    }
  }
  uint32_t prefix = 0, need = a.keep;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    *reinterpret_cast<uint4*>(&sm.count[4 * tid]) = uint4{0u, 0u, 0u, 0u};
    __syncthreads();
    walk(j0, j1, [&](int, uint32_t k, bool on) {
      if (on && (pass == 0 || k >> (shift + bits) == prefix)) atomicAdd(&sm.count[(k >> shift & ((1u << bits) - 1)) * COPIES + (lane & (COPIES - 1))], 1u);
    });
    __syncthreads();
    // thread t: bins 2047 - 2 t and the one below, from the top
    const uint4 v = *reinterpret_cast<const uint4*>(&sm.count[(BINS - 2 - 2 * tid) * COPIES]);
    const uint32_t c[2] = {v.z + v.w, v.x + v.y};
    uint32_t upto = wave_scan(c[0] + c[1]);
    if (lane == 63) sm.in_wave[wave] = upto;
    __syncthreads();
    int all;
    upto += before_wave(sm.in_wave, wave, lane, all);
    uint32_t before = upto - c[0] - c[1];
    if (before < need && need <= upto) {
      const int i = before + c[0] < need;
      if (i) before += c[0];
      sm.found[0] = prefix << bits | (uint32_t)(BINS - 1 - 2 * tid - i);
      sm.found[1] = need - before;
      sm.found[2] = c[i];
    }
    __syncthreads();
    prefix = sm.found[0], need = sm.found[1];
  }
  // kept: keys above `prefix`, and the first `need` of those that are equal to it
  const bool all_equal = sm.found[2] == need;  // every one of those (the usual case: one): no ranks among them
  int ties = 0;
  if (!all_equal) {
    int n_equal = 0;
    walk(j0, j1, [&](int, uint32_t k, bool on) { n_equal += __popcll(__ballot(on && k == prefix)); });
    if (lane == 0) sm.equal[wave] = n_equal;
    __syncthreads();
    int all;
    ties = before_wave(sm.equal, wave, lane, all);
  }
  const uint64_t below = (1ull << lane) - 1;
  // (the ballots of a chunk; `tie`: equal keys before it)
  auto stays = [&](uint32_t k, bool on, int& tie) {
    if (all_equal) return on && k >= prefix;
    const uint64_t same = __ballot(on && k == prefix);
    const bool yes = on && (k > prefix || (k == prefix && tie + __popcll(same & below) < (int)need));
    tie += __popcll(same);
    return yes;
  };
  // the part's slots below keep, of which those not kept become free, and those from there on, of which those kept move
  const int mid = min(max(a.keep, j0), j1);
  int frees = 0, moves = 0, tie = ties;
  if (all_equal) {  // each lane counts, and the wave adds up once
    walk(j0, mid, [&](int, uint32_t k, bool on) { frees += on && k < prefix; });
    walk(mid, j1, [&](int, uint32_t k, bool on) { moves += on && k >= prefix; });
    frees = wave_total(frees), moves = wave_total(moves);
  } else {
    walk(j0, mid, [&](int, uint32_t k, bool on) {  // (stays() in every lane, those behind `mid` too: it counts the equal keys for what follows)
      const bool kept = stays(k, on, tie);
      frees += __popcll(__ballot(on && !kept));
    });
    walk(mid, j1, [&](int, uint32_t k, bool on) { moves += __popcll(__ballot(stays(k, on, tie))); });
  }
  if (lane == 0) sm.n_free[wave] = frees, sm.n_moved[wave] = moves;
  __syncthreads();
  int all;
  int at_moved = before_wave(sm.n_moved, wave, lane, all), at_free = before_wave(sm.n_free, wave, lane, all);
  int32_t* const free = a.free + unit * a.keep;
  int32_t* const moved = a.moved + unit * a.keep;
  int32_t* const src = a.src + unit * a.keep;
  tie = ties;
  walk(j0, mid, [&](int j, uint32_t k, bool on) {
    const bool kept = stays(k, on, tie);
    const uint64_t gone = __ballot(on && !kept);
    if (kept) src[j] = j;
    else if (on) free[at_free + __popcll(gone & below)] = j;
    at_free += __popcll(gone);
  });
  walk(mid, j1, [&](int j, uint32_t k, bool on) {
    const bool kept = stays(k, on, tie);
    const uint64_t go = __ballot(kept);
    const int at = at_moved + __popcll(go & below);
    if (kept && at < a.keep) moved[at] = j;
    at_moved += __popcll(go);
  });
  __threadfence_block();
  __syncthreads();
  all = min(all, a.keep);
  for (int i = tid; i < all; i += CT) {
    const uint32_t to = free[i];
    if (to < (uint32_t)a.keep) src[to] = moved[i];
  }
  __threadfence_block();
  __syncthreads();
  // what a place's mass and position are now: in place those of moved tokens, and positions that were not written down yet
  for (int j = tid; j < a.keep; j += 4 * CT) {
    int from[4], p[4];
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) from[i] = min((uint32_t)src[min(j + CT * i, a.keep - 1)], (uint32_t)tk.ctx - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = tk.mass[from[i]], p[i] = tk.position(from[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int to = j + CT * i;
      if (to >= a.keep || (same_row && from[i] == to && to < tk.kept)) continue;
      if (!same_row || from[i] != to) mass_out[to] = m[i];
      origin_out[to] = p[i];
    }
  }
}

template <int HELD>
__global__ __launch_bounds__(CT) void evict_choose_kernel(Evict a) {
  __shared__ __attribute__((aligned(16))) Counts sm;
  __shared__ uint32_t held[HELD];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int ctx = max(a.lens[b], 0);
  const int64_t r = a.slots[b], ro = a.slots_out[b], unit = (int64_t)b * a.n_kv + h;
  int32_t* head = a.head + unit * 2;
  // (a context that has outgrown its pages or its row stays as it is)
  const bool valid = r >= 0 && r < a.rows && ro >= 0 && ro < a.rows && ctx <= a.cap && ctx <= a.len;
  if (tid == 0) {
    head[0] = !valid ? NOTHING : ctx > a.keep ? LISTED : SAME_PLACES;
    head[1] = ctx;
  }
  if (!valid) return;
  Tokens tk;
  tk.mass = a.mass + (r * a.n_kv + h) * a.len;
  tk.origin = a.origin + (r * a.n_kv + h) * a.len;
  tk.kept = min(a.evicted[2 * r], ctx), tk.dropped = a.evicted[2 * r + 1], tk.ctx = ctx, tk.sinks = a.sinks, tk.recent = a.recent;
  float* mass_out = a.mass + (ro * a.n_kv + h) * a.len;
  int32_t* origin_out = a.origin + (ro * a.n_kv + h) * a.len;
  if (ctx == 0) {
    // No tokens: the pair alone, and only to a row that no other sequence of the call names - rows that a batch is filled up with may name
    // anybody's.  Here and not in the launch that writes the others': nobody reads the row, and the pair read is not written yet.
    if (h != 0 || r == ro) return;
    if (tid == 0) sm.found[0] = 0;
    __syncthreads();
    for (int i = tid; i < (int)gridDim.y; i += CT)
      if (i != b && (a.slots[i] == ro || a.slots_out[i] == ro)) sm.found[0] = 1;
    __syncthreads();
    if (tid == 0 && sm.found[0] == 0) a.evicted[2 * ro] = a.evicted[2 * r], a.evicted[2 * ro + 1] = a.evicted[2 * r + 1];
    return;
  }
  if (ctx <= a.keep) {
    if (r != ro) {
      for (int j = tid; j < ctx; j += CT) mass_out[j] = tk.mass[j];
      for (int j = tid; j < tk.kept; j += CT) origin_out[j] = tk.origin[j];
    }
    return;
  }
  if (ctx <= HELD) choose<true>(a, tk, sm, held, mass_out, origin_out, r == ro, unit);
  else choose<false>(a, tk, sm, held, mass_out, origin_out, r == ro, unit);
}

// lengths and rows, once everything has read the ones before.  (A row that keeps what it has is not written.)
__device__ __forceinline__ void finish(const Evict& a, int b, int mode, int ctx, int n) {
  a.lens_out[b] = mode == NOTHING ? ctx : n;
  if (mode == NOTHING || ctx == 0) return;
  const int64_t r = a.slots[b], ro = a.slots_out[b];
  if (mode == SAME_PLACES && r == ro) return;
  const int kept = a.evicted[2 * r], dropped = a.evicted[2 * r + 1];
  a.evicted[2 * ro] = mode == LISTED ? n : kept;
  a.evicted[2 * ro + 1] = mode == LISTED ? dropped + ctx - n : dropped;
}

// past the caches' own order of replacement: 156 to 139 us for 8 sequences from 32768 tokens, 35 to 28 for 32 back to 4096 (16-byte pieces; single values
// that way take longer, 168 and 40)
__device__ __forceinline__ void store_once(u32x4 v, uint16_t* to) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(to)); }
// of a 16-byte piece of V, which holds two dims (16 apart) of four tokens: dim `hi` of token f % 4
__device__ __forceinline__ uint32_t value(const u32x4& x, int hi, int f) { return (f & 2 ? x[2 * hi + 1] : x[2 * hi]) >> (f & 1) * 16 & 0xffffu; }

// A wave: one tile of 16 places of one kv head; places whose page and slot are the old ones are left.  K goes in the 16-byte pieces that a token is
// in; a piece of V holds four tokens: whole where all four are replaced, else their values one by one (2 bytes; read, patched and written back
// whole: 40 us against 35 for 32 sequences back to 4096 tokens, before store_once).  A token's K is in D / 8 lines of the cache and its V in a quarter of a tile:
// what bounds this is the lines that hold a mover, not the movers' bytes.  (16 lanes for four places, taken from the list of movers, touch the same
// lines: 39 us, 171 against 153 for 8 sequences from 32768 tokens, and 12 against 4 for one from 1100 to 1024; four tiles a wave: 32, 159 and 7;
// all before store_once.  Now 28, 141 and 4.)
template <int DB>
__global__ __launch_bounds__(256) void evict_move_kernel(Evict a) {
  constexpr int TILE = 512 * DB;
  const int h = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 63, t = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int64_t unit = (int64_t)b * a.n_kv + h;
  const int mode = a.head[unit * 2], ctx = a.head[unit * 2 + 1], n = min(ctx, a.keep);
  if (h == 0 && t == 0 && lane == 0) finish(a, b, mode, ctx, n);
  if (mode == NOTHING || 16 * t >= n) return;
  const int g = lane >> 4, c = lane & 15;
  const int32_t *row = a.table + (int64_t)b * a.table_stride, *row_out = a.table_out + (int64_t)b * a.table_out_stride;
  const int to = row_out[t / a.tpb];
  const int slot = 16 * t + c;
  const int from = slot < n && mode == LISTED ? min((uint32_t)a.src[unit * a.keep + slot], (uint32_t)ctx - 1) : slot;
  const int page = slot < n ? row[from / (16 * a.tpb)] : -1;
  const bool moves = slot < n && page >= 0 && page < a.num_blocks && (from != slot || page != to);
  if (to < 0 || to >= a.num_blocks || !__any(moves)) return;
  const int64_t dst = (((int64_t)to * a.n_kv + h) * a.tpb + t % a.tpb) * TILE;
  const int64_t src = moves ? (((int64_t)page * a.n_kv + h) * a.tpb + from / 16 % a.tpb) * TILE : 0;
  if (moves) {
    const uint16_t* p = a.kc + src + (g * 16 + from % 16) * 8;
    u32x4 x[DB];
#pragma unroll
    for (int kk = 0; kk < DB; ++kk) x[kk] = *reinterpret_cast<const u32x4*>(p + kk * 512);
#pragma unroll
    for (int kk = 0; kk < DB; ++kk) store_once(x[kk], a.kc + dst + kk * 512 + (g * 16 + c) * 8);
  }
  u32x4 y[4][DB];
  int f[4];
  bool mv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // token 4 g + e of the tile
    const int who = 4 * g + e;
    mv[e] = __shfl((int)moves, who, 64);
    f[e] = __shfl(from, who, 64);
    const int64_t s = ((int64_t)__shfl((int)(src >> 32), who, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)src, who, 64);
    if (mv[e])
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) y[e][kk] = *reinterpret_cast<const u32x4*>(a.vc + s + kk * 512 + (f[e] % 16 / 4 * 16 + c) * 8);
  }
  uint16_t* const to_v = a.vc + dst + lane * 8;
  if (mv[0] && mv[1] && mv[2] && mv[3]) {
#pragma unroll
    for (int kk = 0; kk < DB; ++kk) {
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[e] = value(y[2 * e][kk], 0, f[2 * e]) | value(y[2 * e + 1][kk], 0, f[2 * e + 1]) << 16;
        v[2 + e] = value(y[2 * e][kk], 1, f[2 * e]) | value(y[2 * e + 1][kk], 1, f[2 * e + 1]) << 16;
      }
      store_once(v, to_v + kk * 512);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (mv[e])
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) {
        to_v[kk * 512 + e] = (uint16_t)value(y[e][kk], 0, f[e]);
        to_v[kk * 512 + 4 + e] = (uint16_t)value(y[e][kk], 1, f[e]);
      }
}

size_t evict_ints(int64_t batch, int64_t n_kv, int64_t keep, int64_t cap) { return batch * n_kv * (2 + (keep < cap ? 3 * keep : 0)); }

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" size_t mi_kv_cache_evict_workspace(int batch, int n_kv_heads, int keep, int block_size, int table_width) {
  if (batch <= 0 || n_kv_heads <= 0 || keep <= 0 || block_size <= 0 || table_width <= 0) return 0;
  return evict_ints(batch, n_kv_heads, keep, (int64_t)block_size * table_width) * 4;
}

extern "C" int mi_kv_cache_evict(mi_bf16* k_cache, mi_bf16* v_cache, int64_t num_blocks, const int32_t* block_table, int64_t table_stride,
                                 const int32_t* block_table_out, int64_t table_out_stride, int table_width, const int32_t* context_lens,
                                 int32_t* context_lens_out, float* mass, int32_t* origin, int32_t* evicted, int64_t mass_rows,
                                 int64_t mass_len, const int32_t* slots, const int32_t* slots_out, int keep, int sinks, int recent,
                                 void* workspace, size_t ws_bytes, int batch, int n_kv_heads, int head_dim, int block_size,
                                 mi_stream stream) {
  if (batch < 0 || n_kv_heads <= 0 || num_blocks <= 0 || table_width <= 0 || table_stride < table_width || table_out_stride < 0 ||
      mass_rows < 0 || mass_len < 0 || block_size <= 0 || keep <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep)
    return MI_EINVAL;
  const int64_t cap = (int64_t)block_size * table_width;
  if ((head_dim != 64 && head_dim != 128) || block_size % 16 != 0 || cap >= (1 << 30) || batch > 65535 || n_kv_heads > 65535) return MI_EUNSUPPORTED;
  if (batch == 0) return MI_OK;
  if (k_cache == nullptr || v_cache == nullptr || block_table == nullptr || block_table_out == nullptr || context_lens == nullptr ||
      context_lens_out == nullptr || mass == nullptr || origin == nullptr || evicted == nullptr || slots == nullptr || slots_out == nullptr ||
      workspace == nullptr)
    return MI_EINVAL;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace)) return MI_EINVAL;
  const int64_t most = std::min<int64_t>(keep, cap), units = (int64_t)batch * n_kv_heads;
  const int64_t blocks = ((most + 15) / 16 + 3) / 4;
  // the places below `most` have pages of their own
  if (table_out_stride < (most + block_size - 1) / block_size) return MI_EINVAL;
  if (blocks > 65535) return MI_EUNSUPPORTED;
  if (ws_bytes < evict_ints(batch, n_kv_heads, keep, cap) * 4) return MI_EWORKSPACE;
  Evict a;
  a.kc = k_cache, a.vc = v_cache, a.num_blocks = num_blocks;
  a.table = block_table, a.table_out = block_table_out, a.table_stride = table_stride, a.table_out_stride = table_out_stride;
  a.tpb = block_size / 16, a.cap = (int)cap, a.n_kv = n_kv_heads;
  a.lens = context_lens, a.lens_out = context_lens_out;
  a.mass = mass, a.origin = origin, a.evicted = evicted, a.rows = mass_rows, a.len = mass_len;
  a.slots = slots, a.slots_out = slots_out, a.keep = keep, a.sinks = sinks, a.recent = recent;
  a.head = static_cast<int32_t*>(workspace);
  a.src = a.head + units * 2, a.free = a.src + units * keep, a.moved = a.free + units * keep;
  const dim3 units_grid(n_kv_heads, batch), grid(n_kv_heads, (unsigned)blocks, batch);
  if (cap <= 8192) evict_choose_kernel<8192><<<units_grid, CT, 0, S(stream)>>>(a);
  else evict_choose_kernel<32768><<<units_grid, CT, 0, S(stream)>>>(a);
  if (head_dim == 128) evict_move_kernel<4><<<grid, 256, 0, S(stream)>>>(a);
  else evict_move_kernel<2><<<grid, 256, 0, S(stream)>>>(a);
  return check_launch();
}
