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
  int32_t *head;               // [batch][n_kv][2]: what the second launch does, tokens
  int32_t *src, *free, *moved; // [batch][n_kv][keep]
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
  __device__ uint32_t key(int j) const {
    const int p = position(j);
    return p < sinks || p >= ctx + dropped - recent ? ~0u : key_of(mass[j]);
  }
};

// One workgroup per (kv head, sequence): the keep-th largest key by four passes of 8 bits over the keys (counts in LDS, a column of its
// own per lane: masses share their leading bits, and lanes that add to one address wait for one another), then the lists in slot order.
constexpr int CT = 1024, CW = CT / 64;

__global__ __launch_bounds__(CT) void evict_choose_kernel(Evict a) {
  __shared__ uint32_t count[256 * 32];
  __shared__ uint32_t total[256];
  __shared__ uint32_t sm_prefix, sm_need;
  __shared__ int sm_more[2 * CW], sm_equal[2 * CW];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ctx = max(a.lens[b], 0);
  const int64_t r = a.slots[b], ro = a.slots_out[b];
  int32_t* head = a.head + ((int64_t)b * a.n_kv + h) * 2;
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
  if (ctx <= a.keep) {
    if (r != ro) {
      for (int j = tid; j < ctx; j += CT) mass_out[j] = tk.mass[j];
      for (int j = tid; j < tk.kept; j += CT) origin_out[j] = tk.origin[j];
    }
    return;
  }

  uint32_t prefix = 0, need = a.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * 32; i += CT) count[i] = 0;
    __syncthreads();
    for (int j = tid; j < ctx; j += CT) {
      const uint32_t k = tk.key(j);
      if (shift == 24 || k >> (shift + 8) == prefix) atomicAdd(&count[((k >> shift) & 255) * 32 + (lane & 31)], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t n = 0;
      for (int i = 0; i < 32; ++i) n += count[tid * 32 + ((i + tid) & 31)];
      total[tid] = n;
    }
    __syncthreads();
    if (wave == 0) {  // lane i: bins 255 - 4 i downwards; the one in which the need-th largest is
      uint32_t c[4], sum = 0;
      for (int i = 0; i < 4; ++i) sum += c[i] = total[255 - 4 * lane - i];
      uint32_t upto = sum;
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
      }
      uint32_t before = upto - sum;
      if (before < need && need <= upto) {
        int i = 0;
        while (before + c[i] < need) before += c[i++];
        sm_prefix = prefix << 8 | (uint32_t)(255 - 4 * lane - i);
        sm_need = need - before;
      }
    }
    __syncthreads();
    prefix = sm_prefix, need = sm_need;
  }
  // kept: keys above `prefix`, and of those equal to it the first `need`.  Wave w counts its part of the slots below keep and its part of
  // those behind, in slot order.
  const int part_lo = ((a.keep + CT - 1) / CT) * 64, part_hi = ((ctx - a.keep + CT - 1) / CT) * 64;
  auto range = [&](int side, int& j0, int& j1) {
    j0 = side ? min(a.keep + wave * part_hi, ctx) : min(wave * part_lo, a.keep);
    j1 = side ? min(j0 + part_hi, ctx) : min(j0 + part_lo, a.keep);
  };
  for (int side = 0; side < 2; ++side) {
    int j0, j1, more = 0, equal = 0;
    range(side, j0, j1);
    for (int j = j0; j < j1; j += 64) {
      const bool on = j + lane < j1;
      const uint32_t k = on ? tk.key(j + lane) : 0;
      more += __popcll(__ballot(on && k > prefix));
      equal += __popcll(__ballot(on && k == prefix));
    }
    if (lane == 0) sm_more[side * CW + wave] = more, sm_equal[side * CW + wave] = equal;
  }
  __syncthreads();
  int32_t* src = a.src + ((int64_t)b * a.n_kv + h) * a.keep;
  int32_t* free = a.free + ((int64_t)b * a.n_kv + h) * a.keep;
  int32_t* moved = a.moved + ((int64_t)b * a.n_kv + h) * a.keep;
  const uint64_t below = (1ull << lane) - 1;
  int n_free = 0;
  for (int side = 0; side < 2; ++side) {
    int j0, j1, equal = 0, listed = 0;
    range(side, j0, j1);
    for (int p = 0; p < side * CW + wave; ++p) {
      const int taken = max(0, min(sm_equal[p], (int)need - equal)) + sm_more[p];
      equal += sm_equal[p];
      const int at = p < CW ? min(p * part_lo, a.keep) : 0;
      if (p >= CW) listed += taken;
      else if (side == 0) listed += min(at + part_lo, a.keep) - at - taken;
    }
    for (int j = j0; j < j1; j += 64) {
      const bool on = j + lane < j1;
      const uint32_t k = on ? tk.key(j + lane) : 0;
      const uint64_t ties = __ballot(on && k == prefix);
      const bool stays = on && (k > prefix || (k == prefix && equal + __popcll(ties & below) < (int)need));
      const bool list = on && (side ? stays : !stays);
      const uint64_t lists = __ballot(list);
      if (side == 0 && on) src[j + lane] = j + lane;
      if (list) (side ? moved : free)[listed + __popcll(lists & below)] = j + lane;
      equal += __popcll(ties);
      listed += __popcll(lists);
    }
    if (side == 0) n_free = listed;
  }
  // all waves' lists, and their number: the last wave of the first side ends with it
  __syncthreads();
  if (wave == CW - 1 && lane == 0) sm_need = (uint32_t)n_free;
  __threadfence_block();
  __syncthreads();
  n_free = (int)sm_need;
  for (int i = tid; i < n_free; i += CT) {
    const int to = free[i], from = moved[i];
    src[to] = from;
    if (r == ro) {
      mass_out[to] = tk.mass[from];
      origin_out[to] = tk.position(from);
    }
  }
  __threadfence_block();
  __syncthreads();
  // the positions of slots at or behind what an earlier eviction left are written down now
  for (int j = tid; j < a.keep; j += CT) {
    const int from = src[j];
    if (r != ro) {
      mass_out[j] = tk.mass[from];
      origin_out[j] = tk.position(from);
    } else if (from == j && j >= tk.kept) {
      origin_out[j] = j + tk.dropped;
    }
  }
}

// A wave: one tile of 16 places of one kv head.  K goes in the 16-byte pieces that a token is in; a piece of V holds four tokens, so that a
// wave builds whole pieces of its tile from those of the tokens that move there and what is there already.
template <int DB>
__global__ __launch_bounds__(256) void evict_move_kernel(Evict a) {
  constexpr int TILE = 512 * DB;
  const int h = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 63, t = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int32_t* head = a.head + ((int64_t)b * a.n_kv + h) * 2;
  const int mode = head[0], ctx = head[1], n = min(ctx, a.keep);
  if (h == 0 && t == 0 && lane == 0) {
    a.lens_out[b] = mode == NOTHING ? ctx : n;
    if (mode != NOTHING) {
      const int64_t r = a.slots[b], ro = a.slots_out[b];
      const int kept = a.evicted[2 * r], dropped = a.evicted[2 * r + 1];
      a.evicted[2 * ro] = mode == LISTED ? n : kept;
      a.evicted[2 * ro + 1] = mode == LISTED ? dropped + ctx - n : dropped;
    }
  }
  if (mode == NOTHING || 16 * t >= n) return;
  const int g = lane >> 4, c = lane & 15;
  const int32_t *row = a.table + (int64_t)b * a.table_stride, *row_out = a.table_out + (int64_t)b * a.table_out_stride;
  const int to = row_out[t / a.tpb];
  const int slot = 16 * t + c;
  const int from = slot < n ? (mode == LISTED ? a.src[((int64_t)b * a.n_kv + h) * a.keep + slot] : slot) : slot;
  const int page = slot < n ? row[from / (16 * a.tpb)] : -1;
  // a page that names no block of the cache is neither read nor written
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
    for (int kk = 0; kk < DB; ++kk) *reinterpret_cast<u32x4*>(a.kc + dst + kk * 512 + (g * 16 + c) * 8) = x[kk];
  }
  u32x4 v[DB];
#pragma unroll
  for (int kk = 0; kk < DB; ++kk) v[kk] = *reinterpret_cast<const u32x4*>(a.vc + dst + kk * 512 + lane * 8);
  bool any = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // token 4 g + e of the tile
    const int who = 4 * g + e;
    const bool mv = __shfl((int)moves, who, 64);
    const int f = __shfl(from, who, 64);
    const int64_t s = ((int64_t)__shfl((int)(src >> 32), who, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)src, who, 64);
    if (mv) {
      any = true;
      const int fe = f % 4;
#pragma unroll
      for (int kk = 0; kk < DB; ++kk) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(a.vc + s + kk * 512 + (f % 16 / 4 * 16 + c) * 8);
        const uint32_t lo = (fe >= 2 ? x[1] : x[0]) >> (fe & 1) * 16 & 0xffffu, hi = (fe >= 2 ? x[3] : x[2]) >> (fe & 1) * 16 & 0xffffu;
        const uint32_t sh = (e & 1) * 16, field = 0xffffu << sh;
        v[kk][e >> 1] = (v[kk][e >> 1] & ~field) | lo << sh;
        v[kk][2 + (e >> 1)] = (v[kk][2 + (e >> 1)] & ~field) | hi << sh;
      }
    }
  }
  if (any)
#pragma unroll
    for (int kk = 0; kk < DB; ++kk) *reinterpret_cast<u32x4*>(a.vc + dst + kk * 512 + lane * 8) = v[kk];
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
  if (!aligned16(k_cache) || !aligned16(v_cache)) return MI_EINVAL;
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
  evict_choose_kernel<<<dim3(n_kv_heads, batch), CT, 0, S(stream)>>>(a);
  const dim3 grid(n_kv_heads, (unsigned)blocks, batch);
  if (head_dim == 128) evict_move_kernel<4><<<grid, 256, 0, S(stream)>>>(a);
  else evict_move_kernel<2><<<grid, 256, 0, S(stream)>>>(a);
  return check_launch();
}
