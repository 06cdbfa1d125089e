// Rows of 8-bit integers as the values they stand for: out = q * scale[row], in bf16 or fp32.
//
// HBM bound: 1 byte read and 2 (4) written per element.  A thread takes 16 columns of four rows at a time, one
// 16-byte load each and 32-byte stores; rows of an output that do not start at 32 bytes are stored by 16, or
// by elements.  13400 x 4096: 31 us (5.4 TB/s), 22600 x 16384: 195 us (5.7 TB/s).
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"

namespace ma {
namespace {

constexpr int kDqThreads = 256;
constexpr int kDqRows = 4;                  // of a thread at a time

// 16 values to a place that is aligned to 32 bytes (wide 2) or 16.
__device__ __forceinline__ void dq_words(char* out, const uint32_t* w, int wide) {
  if (wide == 2) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ void dq_store(uint16_t* out, const float (&v)[16], int wide) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  dq_words(reinterpret_cast<char*>(out), w, wide);
}
__device__ __forceinline__ void dq_store(float* out, const float (&v)[16], int wide) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
  dq_words(reinterpret_cast<char*>(out), w, wide);
  dq_words(reinterpret_cast<char*>(out + 8), w + 8, wide);
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
  let_next_start();
  wait_for_previous();
  const int8_t* __restrict__ q = from_here(q_);
  const float* __restrict__ scale = from_here(scale_);
  T* __restrict__ out = from_here(out_);
  const int chunks = (cols + 15) / 16;
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= chunks) return;
  const int step = gridDim.y * blockDim.y;
  for (int row = blockIdx.y * blockDim.y + threadIdx.y; row < rows; row += kDqRows * step) {
    uint4 v[kDqRows];
    float s[kDqRows];
#pragma unroll
    for (int u = 0; u < kDqRows; ++u)
      if (row + u * step < rows) {
        s[u] = scale[row + u * step];
        const int8_t* from = q + (row + u * step) * q_pitch + c * 16;
        if (c * 16 + 16 <= cols) {
          asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w) : "l"(from) : "memory");
        } else {                             // (what is behind a row's last column may not be there)
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c * 16 + i < cols) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(from[i])) << (8 * (i & 3));
          v[u] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
#pragma unroll
    for (int u = 0; u < kDqRows; ++u) {
      if (row + u * step >= rows) break;
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      float f[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        f[i] = s[u] * static_cast<float>(static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3))));
      T* o = out + (row + u * step) * out_pitch + c * 16;
      if (wide && c * 16 + 16 <= cols) {
        dq_store(o, f, wide);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c * 16 + i < cols) dq_one(o + i, f[i]);
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
  const uint64_t align = a->out | static_cast<uint64_t>(a->out_pitch) * item;
  const int wide = (align & 31u) == 0 ? 2 : (align & 15u) == 0 ? 1 : 0;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return MA_ERR_CUDA;
  // eight CTAs per SM, or as many as there are rows for
  const int gx = (chunks + tx - 1) / tx, need = (a->rows + ty - 1) / ty, room = (8 * sms + gx - 1) / gx;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(need < room ? need : room));
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
