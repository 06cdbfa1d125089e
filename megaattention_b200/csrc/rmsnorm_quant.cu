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
// scale NaN and zeros, so that what is computed from it is NaN too.
//
// HBM bound: 3 bytes per element, 7 with a residual.
#include <cuda_runtime.h>
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
__device__ __forceinline__ uint64_t nq_pair(uint32_t bf16x2) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(bf16x2 << 16), "r"(bf16x2 & 0xffff0000u));
  return r;
}
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

template <int NCH, int T, bool RES>
struct Row {
  long long tok;
  uint4 x[NCH], r[RES ? NCH : 1];

  // The row of `slot`, or of the next slot that has one (tok < 0: there is none left).
  __device__ __forceinline__ void fetch(const NormQuant& p, int* slot, int step, int tid) {
    for (tok = -1; *slot < p.slots && (tok = token_of(p, *slot)) < 0; *slot += step) {}
    if (tok < 0) return;
    const uint16_t* xr = p.x + static_cast<long long>(*slot) * p.x_pitch;
    const uint16_t* rr = RES ? p.res_in + tok * p.res_in_pitch : nullptr;
    const int nchunk = p.hidden >> 3;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      x[k] = c < nchunk ? nq_load(xr + c * 8) : make_uint4(0, 0, 0, 0);
      if (RES) r[k] = c < nchunk ? nq_load(rr + c * 8) : make_uint4(0, 0, 0, 0);
    }
    *slot += step;
  }
};

// CTAs of an SM: four chunks and the next row's need more than 64 registers.
constexpr int threads_of(int T) { return T < 128 ? 256 : T; }
constexpr int ctas_of(int NCH, int T) { return (NCH > 2 ? 512 : 1024) / threads_of(T); }

// T threads on a row (32: every warp of the CTA has a row of its own), NCH chunks of 8 columns each.  The
// next row is on its way while a row is worked on.
template <int NCH, int T, bool RES>
__global__ void __launch_bounds__(threads_of(T), ctas_of(NCH, T))
rmsnorm_quant_kernel(const __grid_constant__ NormQuant arg) {
  constexpr int kRows = T < 128 ? 256 / T : 1;          // rows of a CTA at a time
  __shared__ float s_sum[2][T / 32];
  __shared__ uint32_t s_top[2][T / 32];
  wait_for_previous();
  NormQuant p = arg;
  p.weight = from_here(p.weight);
  const int tid = threadIdx.x % T, lane = threadIdx.x & 31, warp = tid >> 5;
  const int nchunk = p.hidden >> 3, step = gridDim.x * kRows;
  int slot = blockIdx.x * kRows + threadIdx.x / T;
  Row<NCH, T, RES> next;
  next.fetch(p, &slot, step, tid);
  uint4 w[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = tid + k * T;
    w[k] = c < nchunk ? reinterpret_cast<const uint4*>(p.weight)[c] : make_uint4(0, 0, 0, 0);
  }
  const float inv_n = 1.f / static_cast<float>(p.hidden);
  uint32_t turn = 0;
  while (next.tok >= 0) {                               // (the same for all threads of the row)
    const long long tok = next.tok;
    uint4 h[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      h[k] = next.x[k];
      if (RES) {
        const uint4 d = next.r[k];
        h[k] = make_uint4(nq_add(h[k].x, d.x), nq_add(h[k].y, d.y), nq_add(h[k].z, d.z), nq_add(h[k].w, d.w));
      }
    }
    next.fetch(p, &slot, step, tid);
    uint64_t hw[NCH][4], ss2 = 0;                       // (two sums, of even and odd columns)
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      if (RES && c < nchunk) *reinterpret_cast<uint4*>(p.res_out + tok * p.res_out_pitch + c * 8) = h[k];
      const uint32_t hv[4] = {h[k].x, h[k].y, h[k].z, h[k].w}, wv[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t a = nq_pair(hv[i]);
        ss2 = nq_fma(a, a, ss2);
        hw[k][i] = nq_mul(a, nq_pair(wv[i]));
        top = nq_top(top, hw[k][i]);
      }
    }
    const uint2 halves = nq_split(ss2);
    float ss = __uint_as_float(halves.x) + __uint_as_float(halves.y);
    uint32_t top_bits = __float_as_uint(top);           // (order as the values do, NaN above all of them)
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
    top = __uint_as_float(top_bits);
    float scale = top * rsqrtf(ss * inv_n + p.eps) * (1.f / 127.f);
    // (below 2^-119 the factor would overflow: such a row's values are below every scale in use)
    const bool none = top < 1.6e-36f;
    const bool bad = !(top < INFINITY) || !(ss < INFINITY) || (!none && !(scale < INFINITY));
    const uint64_t f2 = nq_both(none || bad ? 0.f : 127.f / top);
    if (none) scale = 0.f;
    if (bad) scale = __int_as_float(0x7fc00000);
    if (tid == 0) p.scale[tok] = scale;
    int8_t* qr = p.q + tok * p.q_pitch;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + k * T;
      if (c < nchunk)
        *reinterpret_cast<uint2*>(qr + c * 8) =
            bad ? make_uint2(0, 0) : make_uint2(nq_bytes(hw[k][0], hw[k][1], f2), nq_bytes(hw[k][2], hw[k][3], f2));
    }
  }
}

template <int NCH, int T>
cudaError_t launch_norm_quant(const NormQuant& p, int sms, cudaStream_t stream) {
  constexpr int threads = threads_of(T);
  const int ctas = (p.slots + threads / T - 1) / (threads / T), room = sms * ctas_of(NCH, T);
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
  if (chunks <= 64) e = ma::launch_norm_quant<2, 32>(p, sms, st);
  else if (chunks <= 128) e = ma::launch_norm_quant<4, 32>(p, sms, st);
  else if (chunks <= 256) e = ma::launch_norm_quant<2, 128>(p, sms, st);
  else if (chunks <= 512) e = ma::launch_norm_quant<2, 256>(p, sms, st);
  else if (chunks <= 1024) e = ma::launch_norm_quant<2, 512>(p, sms, st);
  else e = ma::launch_norm_quant<2, 1024>(p, sms, st);
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
