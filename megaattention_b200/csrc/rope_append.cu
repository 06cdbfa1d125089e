// Rotary position embedding of a step's queries and new keys, with the keys and values appended to the
// paged cache on the way: the producer of a paged layer (fused_prefill.cu reads the pages in place).
//
// Row t of the step belongs to sequence b (cu_q[b] <= t < cu_q[b + 1]) and has position
// p = len_b - (cu_q[b + 1] - t), len_b counting the new keys.  q is rotated into `out`, k rotated into row
// p % 128 of page table[b][p / 128], v copied beside it; rotate-half convention as in rope.cu:
//   out[d] = x[d] cos - x[d + 64] sin,   out[d + 64] = x[d + 64] cos + x[d] sin,   angle = p w_d.
// The angle reaches 1e5 radians and more, where 32 bits resolve 0.004: it is reduced in 64 bits, as turns
// p (w_d / 2 pi) less their nearest integer, and sine and cosine are taken of the remainder.
//
// HBM bound: q is read and written, k and v read and written once.  A warp takes a group of a token's
// heads.  Lane l has dimensions 8 (l % 8) + 0..7 and their partners 64 further on, of head l / 8 of four
// at a time, so that the eight sines and cosines that it needs are the same for every head: it computes
// two of each, and the other lanes of its dimensions the rest.  No shared memory and no barrier.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "append_place.h"
#include "launch.cuh"

namespace ma {
namespace {

constexpr int kRaThreads = 128;

__device__ __forceinline__ float ra_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float ra_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t ra_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

struct RopeAppend {
  const uint16_t *q, *k, *v;
  uint16_t *out, *k_cache, *v_cache;
  const int *cu_q, *lens, *table;
  const float* inv_freq;
  int* dropped;                                   // (may be null)
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, out_tok, out_head, table_pitch;
  int num_batch, rows, H, Hkv, num_pages, width;
  int parts, part_heads;                          // warps of a token, heads of each (a multiple of 4)
};

// The last sequence that starts at or before row t: 32 probes at a time.  (Sequences without new rows
// start where their successor does, so the last one is the one that has the row.)
__device__ __forceinline__ int sequence_of(const int* cu_q, int num_batch, int t, int lane) {
  int lo = 0, n = num_batch;
  while (n > 1) {
    const int at = lane * search_step(n);
    const unsigned before = __ballot_sync(0xffffffffu, at < n && cu_q[lo + (at < n ? at : 0)] <= t);
    search_take(__popc(before), &lo, &n);
  }
  return lo;
}

__global__ void __launch_bounds__(kRaThreads) rope_append_kernel(const __grid_constant__ RopeAppend p) {
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * (kRaThreads / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / p.parts), part = static_cast<int>(unit % p.parts);
  const int* cu_q = from_here(p.cu_q);
  if (t >= p.rows || t >= cu_q[p.num_batch]) return;         // rows behind the last sequence: left alone
  const int b = sequence_of(cu_q, p.num_batch, t, lane);
  const int pos = position_of(t, cu_q[b], cu_q[b + 1], p.lens[b]);
  const int page = page_of(pos, p.table + b * p.table_pitch, p.width, p.num_pages);
  const bool stored = page >= 0;
  if (part == 0 && lane == 0 && !stored && p.dropped) atomicAdd(p.dropped, 1);
  if (pos < 0) return;

  const int sub = lane >> 3, dim = (lane & 7) * 8;
  float c[8], s[8];
  {
    float cs[2], sn[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double turns = static_cast<double>(pos) *
                           (static_cast<double>(p.inv_freq[dim + 2 * sub + i]) * 0.15915494309189533577);
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn[i], &cs[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = __shfl_sync(0xffffffffu, cs[i & 1], (lane & 7) + 8 * (i >> 1));
      s[i] = __shfl_sync(0xffffffffu, sn[i & 1], (lane & 7) + 8 * (i >> 1));
    }
  }
  const long long slot = static_cast<long long>(page) * 128 + (pos & 127);
  const int all = p.H + 2 * p.Hkv, from = part * p.part_heads;
  const int to = min(all, from + p.part_heads);
  for (int h = from + sub; h < to; h += 4) {
    const uint16_t* src;
    uint16_t* dst;
    bool turn = true;
    if (h < p.H) {
      src = p.q + t * p.q_tok + h * p.q_head;
      dst = p.out + t * p.out_tok + h * p.out_head;
    } else {
      if (!stored) continue;
      turn = h < p.H + p.Hkv;
      const int j = turn ? h - p.H : h - p.H - p.Hkv;
      src = turn ? p.k + t * p.k_tok + j * p.k_head : p.v + t * p.v_tok + j * p.v_head;
      dst = (turn ? p.k_cache : p.v_cache) + (slot * p.Hkv + j) * 128;
    }
    uint4 lo = *reinterpret_cast<const uint4*>(src + dim), hi = *reinterpret_cast<const uint4*>(src + dim + 64);
    if (turn) {
      const uint32_t lv[4] = {lo.x, lo.y, lo.z, lo.w}, hv[4] = {hi.x, hi.y, hi.z, hi.w};
      uint32_t ol[4], oh[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a0 = ra_lo(lv[j]), a1 = ra_hi(lv[j]), b0 = ra_lo(hv[j]), b1 = ra_hi(hv[j]);
        ol[j] = ra_pack(a0 * c[2 * j] - b0 * s[2 * j], a1 * c[2 * j + 1] - b1 * s[2 * j + 1]);
        oh[j] = ra_pack(b0 * c[2 * j] + a0 * s[2 * j], b1 * c[2 * j + 1] + a1 * s[2 * j + 1]);
      }
      lo = make_uint4(ol[0], ol[1], ol[2], ol[3]);
      hi = make_uint4(oh[0], oh[1], oh[2], oh[3]);
    }
    *reinterpret_cast<uint4*>(dst + dim) = lo;
    *reinterpret_cast<uint4*>(dst + dim + 64) = hi;
  }
}

}  // namespace
}  // namespace ma

extern "C" int ma_rope_append(const ma_rope_append_args* a, void* stream) {
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->k_cache || !a->v_cache || !a->cu_q ||
      !a->cache_seqlens || !a->page_table || !a->inv_freq)
    return MA_ERR_INVALID;
  if (a->rows < 0 || a->num_batch < 1 || a->H_local <= 0 || a->H_kv <= 0 || a->num_pages < 1 ||
      a->table_width < 1 || a->table_pitch < a->table_width)
    return MA_ERR_INVALID;
  const uint64_t ptrs[] = {a->q, a->k, a->v, a->out, a->k_cache, a->v_cache};
  for (uint64_t p : ptrs)
    if (p & 15u) return MA_ERR_INVALID;                                // 16-byte accesses
  const int64_t strides[] = {a->q_tok, a->q_head, a->k_tok, a->k_head, a->v_tok, a->v_head, a->out_tok, a->out_head};
  for (int64_t s : strides)
    if (s < 0 || (s & 7)) return MA_ERR_INVALID;
  const uint64_t words[] = {a->cu_q, a->cache_seqlens, a->page_table, a->inv_freq, a->dropped};
  for (uint64_t p : words)
    if (p & 3u) return MA_ERR_INVALID;
  if (a->H_local > (1 << 20) || a->H_kv > (1 << 20) || a->rows > (1 << 30)) return MA_ERR_CAPACITY;
  if (a->rows == 0) return MA_OK;
  ma::RopeAppend p{};
  p.q = reinterpret_cast<const uint16_t*>(a->q);
  p.k = reinterpret_cast<const uint16_t*>(a->k);
  p.v = reinterpret_cast<const uint16_t*>(a->v);
  p.out = reinterpret_cast<uint16_t*>(a->out);
  p.k_cache = reinterpret_cast<uint16_t*>(a->k_cache);
  p.v_cache = reinterpret_cast<uint16_t*>(a->v_cache);
  p.cu_q = reinterpret_cast<const int*>(a->cu_q);
  p.lens = reinterpret_cast<const int*>(a->cache_seqlens);
  p.table = reinterpret_cast<const int*>(a->page_table);
  p.inv_freq = reinterpret_cast<const float*>(a->inv_freq);
  p.dropped = reinterpret_cast<int*>(a->dropped);
  p.q_tok = a->q_tok; p.q_head = a->q_head; p.k_tok = a->k_tok; p.k_head = a->k_head;
  p.v_tok = a->v_tok; p.v_head = a->v_head; p.out_tok = a->out_tok; p.out_head = a->out_head;
  p.table_pitch = a->table_pitch;
  p.num_batch = a->num_batch; p.rows = a->rows; p.H = a->H_local; p.Hkv = a->H_kv;
  p.num_pages = a->num_pages; p.width = a->table_width;
  const int groups = (a->H_local + 2 * a->H_kv + 3) / 4;               // of four heads
  const int each = 4;                                                  // groups of a warp
  p.parts = (groups + each - 1) / each;
  p.part_heads = each * 4;
  const long long ctas = (static_cast<long long>(p.rows) * p.parts + ma::kRaThreads / 32 - 1) / (ma::kRaThreads / 32);
  if (ctas > 0x7fffffffLL) return MA_ERR_CAPACITY;
  const cudaError_t e = ma::launch_behind(ma::rope_append_kernel, static_cast<int>(ctas), ma::kRaThreads, 0,
                                          static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
