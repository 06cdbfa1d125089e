// Residual add + RMSNorm with an 8-bit result: integers and one scale per token, the operand of the
// next projection (linear_quant.cu).  Rows are packed, or lie in the fused launch's tile-padded C_sym.
//
//   h = bf16(x + residual)  (the residual stream; h = x without one),   r = rsqrt(mean(h^2) + eps),
//   y = h * r * w,   scale = max|y| / 127,   q = round(y / scale).
//
// r is the same for the whole row, so q = round(h w * 127 / max|h w|) needs no statistic but the
// maximum, and both - the sum of h^2 and the maximum of |h w| - come from one pass and one exchange
// between the warps; h w is exact in fp32 (8-bit by 8-bit significands), the sum is fp32.
// A row of zeros gets scale 0 and zeros; a row whose sum of squares, maximum or scale is not finite gets
// scale NaN and zeros, so that what is computed from it is NaN too.  So does one whose mean + eps is below 2^-126:
// its squares have lost their last bits (down to that, n squares are off by 2^-150 each, 2^-24 of the mean).  A
// row of products below 1.6e-36 counts as zeros, whatever eps.
//
// HBM bound: 3 bytes per element, 7 with a residual.  Device time: 13400 x 4096 28 us (5.8 TB/s, 0.90 of the
// measured copy rate), with a residual 64 us (6.0 TB/s); 22600 x 16384 174 us (6.4 TB/s) and 412 us (6.3 TB/s).
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"

namespace ma {
namespace {

// read once: do not keep in L1 (a plain load: the residual may be updated in place)
__device__ __forceinline__ uint4 nq_load(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// Pairs of fp32 (sm_100 has these operations on two floats).
__device__ __forceinline__ uint64_t nq_join(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t nq_pair(uint32_t bf16x2) { return nq_join(bf16x2 << 16, bf16x2 & 0xffff0000u); }
__device__ __forceinline__ uint64_t nq_both(float v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint2 nq_split(uint64_t v) {
  uint2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(r.x), "=r"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t nq_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t nq_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// bf16(a + b) of two pairs, the sums in fp32
__device__ __forceinline__ uint32_t nq_add(uint32_t a, uint32_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(nq_pair(a)), "l"(nq_pair(b)));
  const uint2 v = nq_split(d);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.x)));
  return r;
}
// max(top, |a|, |b|); a NaN stays
__device__ __forceinline__ float nq_top(float top, uint64_t ab) {
  const uint2 v = nq_split(ab);
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(top), "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)));
  return d;
}
__device__ __forceinline__ float nq_max(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// v * f rounded half to even to integers of |.| <= 127, four in a word: with 1.5 * 2^23 added in the same
// operation a float's last bits are the integer, in two's complement.
__device__ __forceinline__ uint32_t nq_bytes(uint64_t ab, uint64_t cd, uint64_t f) {
  const uint64_t magic = nq_both(12582912.f);
  const uint2 x = nq_split(nq_fma(ab, f, magic)), y = nq_split(nq_fma(cd, f, magic));
  return __byte_perm(__byte_perm(x.x, x.y, 0x0040), __byte_perm(y.x, y.y, 0x0040), 0x5410);
}

struct NormQuant {
  const uint16_t *x, *res_in, *weight;
  uint16_t* res_out;
  int8_t* q;
  float* scale;
  const int *cu_q, *fa_b, *fa_mb;             // (null: packed rows)
  int x_pitch, res_in_pitch, res_out_pitch, q_pitch;
  int slots, hidden;
  float eps;
};

// The token row of a slot, -1 for a padding row of a partial tile.
__device__ __forceinline__ int token_of(const NormQuant& p, int slot) {
  if (!p.cu_q) return slot;
  const int t = slot >> 7;
  const int b = p.fa_b[t], q0 = p.cu_q[b];
  const int row = p.fa_mb[t] * 128 + (slot & 127);
  return row < p.cu_q[b + 1] - q0 ? q0 + row : -1;
}
template <class E>
__device__ __forceinline__ E* at_row(E* base, int row, int pitch) {
  return base + static_cast<long long>(row) * pitch;
}

template <int NCH, int T, bool RES>
struct Row {
  int tok;
  uint4 x[NCH], r[RES ? NCH : 1];             // (zeros where the row has no columns)

  // The row of `slot`, or of the next slot that has one (tok < 0: there is none left).
  __device__ __forceinline__ void fetch(const NormQuant& p, int* slot, int step, int tid, int nchunk) {
    for (tok = -1; *slot < p.slots && (tok = token_of(p, *slot)) < 0; *slot += step) {}
    if (tok < 0) return;
    const uint16_t* xr = at_row(p.x, *slot, p.x_pitch) + tid * 8;
    const uint16_t* rr = RES ? at_row(p.res_in, tok, p.res_in_pitch) + tid * 8 : nullptr;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      if (tid + k * T < nchunk) {
        x[k] = nq_load(xr + k * T * 8);
        if (RES) r[k] = nq_load(rr + k * T * 8);
      }
    *slot += step;
  }
};

// CTAs of T threads (32: of 256, a row to each warp), as many as registers allow: 85 a thread with four
// chunks and no residual, 128 with a residual or eight chunks; 64 KB are on their way to an SM then.
constexpr int threads_of(int T) { return T == 32 ? 256 : T; }
constexpr int ctas_of(int NCH, int T, bool RES) { return (NCH > 4 || (RES && NCH > 2) ? 512 : NCH > 2 ? 768 : 1024) / threads_of(T); }

// T threads on a row, NCH chunks of 8 columns each; the next row is on its way while a row is worked on.
// Without a residual there is half as much to load and the instructions count: 15.8 of them per element
// kept 73 % of the issue slots busy at 4.5 TB/s (now 9.9, 66 %, 5.8 TB/s).  So what a row costs beside its
// columns is spread over four to eight chunks a thread, the weights lie in shared memory, as fp32 where they
// fit, and pitches are 32 bits.
template <int NCH, int T, bool RES>
__global__ void __launch_bounds__(threads_of(T), ctas_of(NCH, T, RES))
rmsnorm_quant_kernel(const __grid_constant__ NormQuant p) {
  constexpr int kWarps = T / 32, kPad = kWarps < 4 ? 4 : kWarps;
  __shared__ __align__(16) float s_sum[2][kPad], s_top[2][kPad];
  constexpr bool kFull = !RES && NCH * T <= 1024;       // weights as fp32 (bf16 where they are too many)
  __shared__ uint4 s_weight[NCH * T * (kFull ? 2 : 1)];
  let_next_start();
  wait_for_previous();
  const int tid = threadIdx.x % T, lane = threadIdx.x & 31, warp = tid >> 5;
  const int nchunk = p.hidden >> 3, rows = blockDim.x / T, step = gridDim.x * rows;
  int slot = blockIdx.x * rows + threadIdx.x / T;
  Row<NCH, T, RES> next;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    next.x[k] = make_uint4(0, 0, 0, 0);
    if (RES) next.r[k] = make_uint4(0, 0, 0, 0);
  }
  next.fetch(p, &slot, step, tid, nchunk);
  const uint16_t* weight = from_here(p.weight);
  for (int c = threadIdx.x; c < NCH * T; c += blockDim.x) {
    const uint4 w = c < nchunk ? reinterpret_cast<const uint4*>(weight)[c] : make_uint4(0, 0, 0, 0);
    if (kFull) {
      s_weight[c] = make_uint4(w.x << 16, w.x & 0xffff0000u, w.y << 16, w.y & 0xffff0000u);
      s_weight[NCH * T + c] = make_uint4(w.z << 16, w.z & 0xffff0000u, w.w << 16, w.w & 0xffff0000u);
    } else {
      s_weight[c] = w;
    }
  }
  __syncthreads();
  const float inv_n = 1.f / static_cast<float>(p.hidden);
  uint32_t turn = 0;
  while (next.tok >= 0) {                               // (the same for all threads of the row)
    const int tok = next.tok;
    uint4 h[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      h[k] = next.x[k];
      if (RES) {
        const uint4 d = next.r[k];
        h[k] = make_uint4(nq_add(h[k].x, d.x), nq_add(h[k].y, d.y), nq_add(h[k].z, d.z), nq_add(h[k].w, d.w));
      }
    }
    next.fetch(p, &slot, step, tid, nchunk);
    uint64_t hw[NCH][4], ss2 = 0;                       // (two sums, of even and odd columns)
    float top = 0.f;
    uint16_t* ro = RES ? at_row(p.res_out, tok, p.res_out_pitch) + tid * 8 : nullptr;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      if (RES && c < nchunk) *reinterpret_cast<uint4*>(ro + k * T * 8) = h[k];
      const uint32_t hv[4] = {h[k].x, h[k].y, h[k].z, h[k].w};
      const uint4 w0 = s_weight[c], w1 = s_weight[kFull ? NCH * T + c : c];
      const uint64_t wv[4] = {kFull ? nq_join(w0.x, w0.y) : nq_pair(w0.x), kFull ? nq_join(w0.z, w0.w) : nq_pair(w0.y),
                              kFull ? nq_join(w1.x, w1.y) : nq_pair(w0.z), kFull ? nq_join(w1.z, w1.w) : nq_pair(w0.w)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t a = nq_pair(hv[i]);
        ss2 = nq_fma(a, a, ss2);
        hw[k][i] = nq_mul(a, wv[i]);
        top = nq_top(top, hw[k][i]);
      }
    }
    const uint2 halves = nq_split(ss2);
    float ss = __uint_as_float(halves.x) + __uint_as_float(halves.y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    // (the bits of what is not negative order as the values do, NaN above all of them)
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if (T > 32) {
      const uint32_t at = turn & 1u;                    // two buffers: one barrier per row
      ++turn;
      if (lane == 0) { s_sum[at][warp] = ss; s_top[at][warp] = top; }
      __syncthreads();
      ss = 0.f;
      top = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(&s_sum[at][i]);
        const float4 b = *reinterpret_cast<const float4*>(&s_top[at][i]);
        ss += kWarps < 4 ? a.x + a.y : (a.x + a.y) + (a.z + a.w);
        top = nq_max(top, b.x, b.y);
        if (kWarps >= 4) top = nq_max(top, b.z, b.w);
      }
    }
    const float mean = ss * inv_n + p.eps;
    const float scale = top * rsqrtf(mean) * (1.f / 127.f);
    // (below 2^-119 the factor would overflow: such a row's values are below every scale in use)
    const bool none = top < 1.6e-36f;
    const bool bad = !(top < INFINITY) || !(ss < INFINITY) || (!none && !(mean >= FLT_MIN && scale < INFINITY));
    const uint64_t f2 = nq_both(none || bad ? 0.f : 127.f / top);
    if (tid == 0) p.scale[tok] = bad ? __int_as_float(0x7fc00000) : none ? 0.f : scale;
    int8_t* qr = at_row(p.q, tok, p.q_pitch) + tid * 8;
    if (bad) {                                          // (a product with a NaN or an infinity would not be zero)
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        for (int i = 0; i < 4; ++i) hw[k][i] = 0;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      if (tid + k * T < nchunk)
        *reinterpret_cast<uint2*>(qr + k * T * 8) =
            make_uint2(nq_bytes(hw[k][0], hw[k][1], f2), nq_bytes(hw[k][2], hw[k][3], f2));
  }
}

template <int NCH, int T, bool RES>
cudaError_t launch_norm_quant(const NormQuant& p, int sms, cudaStream_t stream) {
  constexpr int threads = threads_of(T);
  const int ctas = (p.slots + threads / T - 1) / (threads / T), room = sms * ctas_of(NCH, T, RES);
  return launch_behind(rmsnorm_quant_kernel<NCH, T, RES>, ctas < room ? ctas : room, threads, 0, stream, p);
}

}  // namespace
}  // namespace ma

extern "C" int ma_rmsnorm_quant(const ma_rmsnorm_quant_args* a, void* stream) {
  if (!a || !a->x || !a->weight || !a->q_out || !a->scale_out) return MA_ERR_INVALID;
  if (!a->residual_in != !a->residual_out) return MA_ERR_INVALID;
  const bool tiles = a->cu_q || a->fa_b || a->fa_mb;
  if (tiles && (!a->cu_q || !a->fa_b || !a->fa_mb)) return MA_ERR_INVALID;
  if (a->rows < 0 || a->hidden <= 0 || (a->hidden & 7) || !(a->eps >= 0.f)) return MA_ERR_INVALID;
  if (a->hidden > 4 * 512 * 8) return MA_ERR_CAPACITY;                 // 16384 columns
  if (a->rows > (tiles ? 1 << 23 : 1 << 30)) return MA_ERR_CAPACITY;   // slots are counted in 32 bits
  if (a->x_pitch < a->hidden || (a->x_pitch & 7) || a->q_pitch < a->hidden || (a->q_pitch & 15))
    return MA_ERR_INVALID;
  if (a->residual_in && (a->residual_in_pitch < a->hidden || (a->residual_in_pitch & 7) ||
                         a->residual_out_pitch < a->hidden || (a->residual_out_pitch & 7)))
    return MA_ERR_INVALID;
  const int64_t pitches[] = {a->x_pitch, a->residual_in_pitch, a->residual_out_pitch, a->q_pitch};
  for (int64_t p : pitches)
    if (p > 0x7ffffff0) return MA_ERR_CAPACITY;
  const uint64_t ptrs[] = {a->x, a->residual_in, a->weight, a->residual_out, a->q_out};
  for (uint64_t p : ptrs)
    if (p & 15u) return MA_ERR_INVALID;                                // 16-byte accesses
  if (a->scale_out & 3u) return MA_ERR_INVALID;
  if (a->rows == 0) return MA_OK;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return MA_ERR_CUDA;
  ma::NormQuant p{};
  p.x = reinterpret_cast<const uint16_t*>(a->x);
  p.res_in = reinterpret_cast<const uint16_t*>(a->residual_in);
  p.weight = reinterpret_cast<const uint16_t*>(a->weight);
  p.res_out = reinterpret_cast<uint16_t*>(a->residual_out);
  p.q = reinterpret_cast<int8_t*>(a->q_out);
  p.scale = reinterpret_cast<float*>(a->scale_out);
  p.cu_q = reinterpret_cast<const int*>(a->cu_q);
  p.fa_b = reinterpret_cast<const int*>(a->fa_b);
  p.fa_mb = reinterpret_cast<const int*>(a->fa_mb);
  p.x_pitch = static_cast<int>(a->x_pitch); p.res_in_pitch = static_cast<int>(a->residual_in_pitch);
  p.res_out_pitch = static_cast<int>(a->residual_out_pitch); p.q_pitch = static_cast<int>(a->q_pitch);
  p.slots = tiles ? a->rows * 128 : a->rows;
  p.hidden = a->hidden; p.eps = a->eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int chunks = a->hidden / 8;
  cudaError_t e;
  if (a->residual_in) {
    if (chunks <= 64) e = ma::launch_norm_quant<2, 32, true>(p, sms, st);
    else if (chunks <= 128) e = ma::launch_norm_quant<4, 32, true>(p, sms, st);
    else if (chunks <= 256) e = ma::launch_norm_quant<4, 64, true>(p, sms, st);
    else if (chunks <= 512) e = ma::launch_norm_quant<4, 128, true>(p, sms, st);
    else if (chunks <= 1024) e = ma::launch_norm_quant<4, 256, true>(p, sms, st);
    else e = ma::launch_norm_quant<4, 512, true>(p, sms, st);
  } else {
    if (chunks <= 64) e = ma::launch_norm_quant<2, 32, false>(p, sms, st);
    else if (chunks <= 128) e = ma::launch_norm_quant<4, 32, false>(p, sms, st);
    else if (chunks <= 256) e = ma::launch_norm_quant<4, 64, false>(p, sms, st);
    else if (chunks <= 512) e = ma::launch_norm_quant<4, 128, false>(p, sms, st);
    else if (chunks <= 1024) e = ma::launch_norm_quant<4, 256, false>(p, sms, st);
    else e = ma::launch_norm_quant<8, 256, false>(p, sms, st);
  }
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
