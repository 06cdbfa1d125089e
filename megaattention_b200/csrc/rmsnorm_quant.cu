// Residual add + RMSNorm with an 8-bit result: integers and one scale per token, the operand of the
// next projection (linear_quant.cu).  Rows are packed, or lie in the fused launch's tile-padded C_sym.
//
//   h = bf16(x + residual)  (the residual stream; h = x without one),   r = rsqrt(mean(h^2) + eps),
//   y = h * r * w,   scale = max|y| / 127,   q = round(y / scale).
//
// r is the same for the whole row, so q = round(h w * 127 / max|h w|) needs no statistic but the
// maximum, and both - the sum of h^2 and the maximum of |h w| - come from one pass and one exchange
// between the warps; h w is exact in fp32 (8-bit by 8-bit significands), the sum is fp32.  The maximum is
// taken over the magnitudes' bit patterns: they order as the values do, and a NaN is above all of them.
// A row of zeros gets scale 0 and zeros; a row whose sum of squares, maximum or scale is not finite gets
// scale NaN and zeros, so that what is computed from it is NaN too.
//
// HBM bound: 3 bytes per element, 7 with a residual.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"

namespace ma {
namespace {

__device__ __forceinline__ float nq_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float nq_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t nq_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// read once: do not keep in L1 (a plain load: the residual may be updated in place)
__device__ __forceinline__ uint4 nq_load(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// Four integers in a word, rounded half to even; |v| <= 127 up to its last bit.
__device__ __forceinline__ uint32_t nq_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040);
  const uint32_t cd = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

struct NormQuant {
  const uint16_t *x, *res_in, *weight;
  uint16_t* res_out;
  int8_t* q;
  float* scale;
  const int *cu_q, *fa_b, *fa_mb;             // (null: packed rows)
  long long x_pitch, res_in_pitch, res_out_pitch, q_pitch;
  int slots, hidden;
  float eps;
};

// The token row of a slot, -1 for a padding row of a partial tile.
__device__ __forceinline__ long long token_of(const NormQuant& p, int slot) {
  if (!p.cu_q) return slot;
  const int t = slot >> 7;
  const int b = p.fa_b[t], q0 = p.cu_q[b];
  const int row = p.fa_mb[t] * 128 + (slot & 127);
  return row < p.cu_q[b + 1] - q0 ? q0 + row : -1;
}

// T threads on a row (32: every warp of the CTA has a row of its own), NCH chunks of 8 columns each.
template <int NCH, int T, bool RES>
__global__ void __launch_bounds__(T < 256 ? 256 : T, 1024 / (T < 256 ? 256 : T))
rmsnorm_quant_kernel(const __grid_constant__ NormQuant arg) {
  constexpr int kRows = T < 256 ? 256 / T : 1;          // rows of a CTA at a time
  __shared__ float s_sum[2][T / 32];
  __shared__ uint32_t s_top[2][T / 32];
  wait_for_previous();
  NormQuant p = arg;
  p.weight = from_here(p.weight);
  const int tid = threadIdx.x % T, lane = threadIdx.x & 31, warp = tid >> 5;
  const int nchunk = p.hidden >> 3;
  uint4 w[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = tid + k * T;
    w[k] = c < nchunk ? reinterpret_cast<const uint4*>(p.weight)[c] : make_uint4(0, 0, 0, 0);
  }
  const float inv_n = 1.f / static_cast<float>(p.hidden);
  uint32_t turn = 0;
  for (int slot = blockIdx.x * kRows + threadIdx.x / T; slot < p.slots; slot += gridDim.x * kRows) {
    const long long tok = token_of(p, slot);
    if (tok < 0) continue;                              // (the same for all threads of the row)
    const uint16_t* xr = p.x + static_cast<long long>(slot) * p.x_pitch;
    uint4 h[NCH];
    float ss = 0.f;
    uint32_t top_bits = 0;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      h[k] = c < nchunk ? nq_load(xr + c * 8) : make_uint4(0, 0, 0, 0);
    }
    if (RES) {
      const uint16_t* rr = p.res_in + tok * p.res_in_pitch;
      uint16_t* ro = p.res_out + tok * p.res_out_pitch;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int c = tid + k * T;
        if (c < nchunk) {
          const uint4 d = nq_load(rr + c * 8);
          h[k].x = nq_pack(nq_lo(h[k].x) + nq_lo(d.x), nq_hi(h[k].x) + nq_hi(d.x));
          h[k].y = nq_pack(nq_lo(h[k].y) + nq_lo(d.y), nq_hi(h[k].y) + nq_hi(d.y));
          h[k].z = nq_pack(nq_lo(h[k].z) + nq_lo(d.z), nq_hi(h[k].z) + nq_hi(d.z));
          h[k].w = nq_pack(nq_lo(h[k].w) + nq_lo(d.w), nq_hi(h[k].w) + nq_hi(d.w));
          *reinterpret_cast<uint4*>(ro + c * 8) = h[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const uint32_t hv[4] = {h[k].x, h[k].y, h[k].z, h[k].w}, wv[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = nq_lo(hv[i]), b = nq_hi(hv[i]);
        ss = fmaf(a, a, ss);
        ss = fmaf(b, b, ss);
        top_bits = max(top_bits, __float_as_uint(a * nq_lo(wv[i])) & 0x7fffffffu);
        top_bits = max(top_bits, __float_as_uint(b * nq_hi(wv[i])) & 0x7fffffffu);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    top_bits = __reduce_max_sync(0xffffffffu, top_bits);
    if (T > 32) {
      const uint32_t at = turn & 1u;                    // two buffers: one barrier per row
      ++turn;
      if (lane == 0) { s_sum[at][warp] = ss; s_top[at][warp] = top_bits; }
      __syncthreads();
      ss = 0.f;
      top_bits = 0;
#pragma unroll
      for (int i = 0; i < T / 32; ++i) { ss += s_sum[at][i]; top_bits = max(top_bits, s_top[at][i]); }
    }
    const float top = __uint_as_float(top_bits);
    float scale = top * rsqrtf(ss * inv_n + p.eps) * (1.f / 127.f);
    // (below 2^-119 the factor would overflow: such a row's values are below every scale in use)
    const bool none = top < 1.6e-36f;
    const bool bad = !(top < INFINITY) || !(ss < INFINITY) || (!none && !(scale < INFINITY));
    const float f = none || bad ? 0.f : 127.f / top;
    if (none) scale = 0.f;
    if (bad) scale = __int_as_float(0x7fc00000);
    if (tid == 0) p.scale[tok] = scale;
    int8_t* qr = p.q + tok * p.q_pitch;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      if (c < nchunk) {
        const uint32_t hv[4] = {h[k].x, h[k].y, h[k].z, h[k].w}, wv[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
        uint32_t o[2] = {0, 0};
        if (!bad) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            o[i] = nq_bytes(nq_lo(hv[2 * i]) * nq_lo(wv[2 * i]) * f, nq_hi(hv[2 * i]) * nq_hi(wv[2 * i]) * f,
                            nq_lo(hv[2 * i + 1]) * nq_lo(wv[2 * i + 1]) * f,
                            nq_hi(hv[2 * i + 1]) * nq_hi(wv[2 * i + 1]) * f);
        }
        *reinterpret_cast<uint2*>(qr + c * 8) = make_uint2(o[0], o[1]);
      }
    }
  }
}

template <int NCH, int T>
cudaError_t launch_norm_quant(const NormQuant& p, int sms, cudaStream_t stream) {
  constexpr int threads = T < 256 ? 256 : T;
  const int ctas = (p.slots + threads / T - 1) / (threads / T), room = sms * (1024 / threads);
  const int grid = ctas < room ? ctas : room;
  if (p.res_in) return launch_behind(rmsnorm_quant_kernel<NCH, T, true>, grid, threads, 0, stream, p);
  return launch_behind(rmsnorm_quant_kernel<NCH, T, false>, grid, threads, 0, stream, p);
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
  p.x_pitch = a->x_pitch; p.res_in_pitch = a->residual_in_pitch;
  p.res_out_pitch = a->residual_out_pitch; p.q_pitch = a->q_pitch;
  p.slots = tiles ? a->rows * 128 : a->rows;
  p.hidden = a->hidden; p.eps = a->eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int chunks = a->hidden / 8;
  cudaError_t e;
  if (chunks <= 128) e = ma::launch_norm_quant<4, 32>(p, sms, st);
  else if (chunks <= 256) e = ma::launch_norm_quant<1, 256>(p, sms, st);
  else if (chunks <= 512) e = ma::launch_norm_quant<2, 256>(p, sms, st);
  else if (chunks <= 1024) e = ma::launch_norm_quant<4, 256>(p, sms, st);
  else e = ma::launch_norm_quant<4, 512>(p, sms, st);
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
