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
// HBM bound: q is read and written, k and v read and written once.  22600 tokens of 64 + 8 heads: 143 us, 6.46
// TB/s, the measured copy rate; 1384 tokens of 16 + 2 heads 4.8 us (7.4 with the place looked up before the
// first load), 64 tokens of 8 + 1 heads 3.0.  A warp takes sixteen of a token's heads.  Lane l has
// dimensions 8 (l % 8) + 0..7 and their partners 64 further on, of head l / 8 of four at a time, so that the
// eight sines and cosines that it needs are the same for every head: it computes two of each, and the other
// lanes of its dimensions the rest.  No shared memory and no barrier.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "append_place.h"
#include "launch.cuh"

namespace ma {
namespace {

constexpr int kRaThreads = 128;
constexpr int kRaGroups = 4;                      // groups of four heads of a warp

__device__ __forceinline__ float ra_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float ra_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t ra_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// read once; the asm keeps its place before the look-up
__device__ __forceinline__ uint4 ra_load(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

struct RopeAppend {
  const uint16_t *q, *k, *v;
  uint16_t *out, *k_cache, *v_cache;
  const int *cu_q, *lens, *table;
  const float* inv_freq;
  int* dropped;                                   // (may be null)
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, out_tok, out_head, table_pitch;
  int num_batch, rows, H, Hkv, num_pages, width;
  int parts;                                      // warps of a token
};

struct Place {
  int pos, page;                                  // -1: none
};

// Where row t goes.  The sequence is the last one that starts at or before the row, looked for with 32
// probes at a time (sequences without new rows start where their successor does, so the last one is the one
// that has the row).  A batch that fits a warp takes lengths along with the starts: one trip to memory less
// before the page is known.
__device__ __forceinline__ Place place_of(const RopeAppend& p, const int* cu_q, int t, int lane) {
  Place at;
  int b = 0, q0, q1, len;
  if (p.num_batch <= kSmallBatch) {
    const int start = cu_q[small_start(lane, p.num_batch)], n = p.lens[small_keys(lane, p.num_batch)];
    b = small_take(__popc(__ballot_sync(0xffffffffu, lane < p.num_batch && start <= t)));
    q0 = __shfl_sync(0xffffffffu, start, b);
    q1 = __shfl_sync(0xffffffffu, start, b + 1);
    len = __shfl_sync(0xffffffffu, n, b);
  } else {
    int n = p.num_batch;
    while (n > 1) {
      const int i = lane * search_step(n);
      const unsigned before = __ballot_sync(0xffffffffu, i < n && cu_q[b + (i < n ? i : 0)] <= t);
      search_take(__popc(before), &b, &n);
    }
    q0 = cu_q[b];
    q1 = cu_q[b + 1];
    len = p.lens[b];
  }
  at.pos = position_of(t, q0, q1, len);
  at.page = page_of(at.pos, p.table + b * p.table_pitch, p.width, p.num_pages);
  return at;
}

__global__ void __launch_bounds__(kRaThreads) rope_append_kernel(const __grid_constant__ RopeAppend p) {
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * (kRaThreads / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / p.parts), part = static_cast<int>(unit % p.parts);
  if (t >= p.rows) return;
  const int* cu_q = from_here(p.cu_q);
  const int sub = lane >> 3, dim = (lane & 7) * 8;
  const int first = part * (4 * kRaGroups) + sub, all = p.H + 2 * p.Hkv;

  // What this lane takes from its heads is on its way (rows behind the last sequence are the caller's too)
  // while the row's place is looked up.
  uint4 lo[kRaGroups], hi[kRaGroups];
#pragma unroll
  for (int g = 0; g < kRaGroups; ++g) {
    const int h = first + 4 * g;
    if (h >= all) break;
    const int j = h < p.H ? h : h - p.H < p.Hkv ? h - p.H : h - p.H - p.Hkv;
    const uint16_t* src = h < p.H ? p.q + t * p.q_tok + j * p.q_head
                                  : h - p.H < p.Hkv ? p.k + t * p.k_tok + j * p.k_head : p.v + t * p.v_tok + j * p.v_head;
    lo[g] = ra_load(src + dim);
    hi[g] = ra_load(src + dim + 64);
  }
  if (t >= cu_q[p.num_batch]) return;              // rows behind the last sequence: left alone
  const Place at = place_of(p, cu_q, t, lane);
  if (part == 0 && lane == 0 && at.page < 0 && p.dropped) atomicAdd(p.dropped, 1);
  if (at.pos < 0) return;

  float c[8], s[8];
  {
    float cs[2], sn[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double turns = static_cast<double>(at.pos) *
                           (static_cast<double>(p.inv_freq[dim + 2 * sub + i]) * 0.15915494309189533577);
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn[i], &cs[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = __shfl_sync(0xffffffffu, cs[i & 1], (lane & 7) + 8 * (i >> 1));
      s[i] = __shfl_sync(0xffffffffu, sn[i & 1], (lane & 7) + 8 * (i >> 1));
    }
  }
  const long long slot = static_cast<long long>(at.page) * 128 + (at.pos & 127);
#pragma unroll
  for (int g = 0; g < kRaGroups; ++g) {
    const int h = first + 4 * g;
    if (h >= all) break;
    uint16_t* dst = p.out + t * p.out_tok + h * p.out_head;
    const bool turn = h < p.H + p.Hkv;
    if (h >= p.H) {
      if (at.page < 0) break;
      dst = (turn ? p.k_cache : p.v_cache) + (slot * p.Hkv + (turn ? h - p.H : h - p.H - p.Hkv)) * 128;
    }
    if (turn) {
      const uint32_t lv[4] = {lo[g].x, lo[g].y, lo[g].z, lo[g].w}, hv[4] = {hi[g].x, hi[g].y, hi[g].z, hi[g].w};
      uint32_t ol[4], oh[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a0 = ra_lo(lv[j]), a1 = ra_hi(lv[j]), b0 = ra_lo(hv[j]), b1 = ra_hi(hv[j]);
        ol[j] = ra_pack(a0 * c[2 * j] - b0 * s[2 * j], a1 * c[2 * j + 1] - b1 * s[2 * j + 1]);
        oh[j] = ra_pack(b0 * c[2 * j] + a0 * s[2 * j], b1 * c[2 * j + 1] + a1 * s[2 * j + 1]);
      }
      lo[g] = make_uint4(ol[0], ol[1], ol[2], ol[3]);
      hi[g] = make_uint4(oh[0], oh[1], oh[2], oh[3]);
    }
    *reinterpret_cast<uint4*>(dst + dim) = lo[g];
    *reinterpret_cast<uint4*>(dst + dim + 64) = hi[g];
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
  p.parts = (a->H_local + 2 * a->H_kv + 4 * ma::kRaGroups - 1) / (4 * ma::kRaGroups);
  const long long ctas = (static_cast<long long>(p.rows) * p.parts + ma::kRaThreads / 32 - 1) / (ma::kRaThreads / 32);
  if (ctas > 0x7fffffffLL) return MA_ERR_CAPACITY;
  const cudaError_t e = ma::launch_behind(ma::rope_append_kernel, static_cast<int>(ctas), ma::kRaThreads, 0,
                                          static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
