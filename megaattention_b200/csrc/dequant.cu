// Rows of 8-bit integers as the values they stand for: out = q * scale[row], in bf16 or fp32.
//
// HBM bound: 1 byte read and 2 (4) written per element.  A thread takes 16 columns, one 16-byte load and
// two (four) 16-byte stores; rows of an output that does not start at 16 bytes are stored by elements.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"

namespace ma {
namespace {

constexpr int kDqThreads = 256;

__device__ __forceinline__ void dq_store(uint16_t* out, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void dq_store(float* out, const float (&v)[8]) {
  reinterpret_cast<float4*>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void dq_one(uint16_t* out, float v) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(0.f), "f"(v));
  *out = static_cast<uint16_t>(w);
}
__device__ __forceinline__ void dq_one(float* out, float v) { *out = v; }

template <typename T>
__global__ void __launch_bounds__(kDqThreads)
dequant_kernel(const int8_t* q_, const float* scale_, T* out_, long long q_pitch, long long out_pitch, int rows,
               int cols, int wide) {
  wait_for_previous();
  const int8_t* __restrict__ q = from_here(q_);
  const float* __restrict__ scale = from_here(scale_);
  T* __restrict__ out = from_here(out_);
  const int chunks = (cols + 15) / 16;
  for (int row = blockIdx.y * blockDim.y + threadIdx.y; row < rows; row += gridDim.y * blockDim.y) {
    const float s = scale[row];
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += gridDim.x * blockDim.x) {
      const uint4 v = *reinterpret_cast<const uint4*>(q + row * q_pitch + c * 16);    // (rows are 16-byte multiples)
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      T* o = out + row * out_pitch + c * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          f[i] = s * static_cast<float>(static_cast<int8_t>(w[2 * h + (i >> 2)] >> (8 * (i & 3))));
        if (wide && c * 16 + 8 * h + 8 <= cols) {
          dq_store(o + 8 * h, f);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c * 16 + 8 * h + i < cols) dq_one(o + 8 * h + i, f[i]);
        }
      }
    }
  }
}

}  // namespace
}  // namespace ma

extern "C" int ma_dequant(const ma_dequant_args* a, void* stream) {
  if (!a || !a->q || !a->scale || !a->out) return MA_ERR_INVALID;
  const int item = a->out_f32 ? 4 : 2;
  if (a->rows < 0 || a->cols < 0 || a->q_pitch < a->cols || (a->q_pitch & 15) || a->out_pitch < a->cols)
    return MA_ERR_INVALID;
  if ((a->q & 15u) || (a->scale & 3u) || (a->out & (item - 1u))) return MA_ERR_INVALID;
  if (a->rows > (1 << 30) || a->cols > (1 << 30)) return MA_ERR_CAPACITY;
  if (a->rows == 0 || a->cols == 0) return MA_OK;
  // the threads of a CTA lie along the columns as far as there are any
  int tx = 1;
  const int chunks = (a->cols + 15) / 16;
  while (tx < chunks && tx < ma::kDqThreads) tx *= 2;
  const int ty = ma::kDqThreads / tx;
  const int wide = (a->out & 15u) == 0 && (a->out_pitch * item & 15) == 0;
  const dim3 grid(static_cast<unsigned>((chunks + tx - 1) / tx),
                  static_cast<unsigned>((a->rows + ty - 1) / ty < 32768 ? (a->rows + ty - 1) / ty : 32768));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(tx), static_cast<unsigned>(ty));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int8_t* q = reinterpret_cast<const int8_t*>(a->q);
  const float* scale = reinterpret_cast<const float*>(a->scale);
  const long long qp = a->q_pitch, op = a->out_pitch;
  const cudaError_t e =
      a->out_f32 ? cudaLaunchKernelEx(&cfg, ma::dequant_kernel<float>, q, scale, reinterpret_cast<float*>(a->out), qp,
                                      op, a->rows, a->cols, wide)
                 : cudaLaunchKernelEx(&cfg, ma::dequant_kernel<uint16_t>, q, scale,
                                      reinterpret_cast<uint16_t*>(a->out), qp, op, a->rows, a->cols, wide);
  const cudaError_t last = cudaGetLastError();
  return e == cudaSuccess && last == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}
