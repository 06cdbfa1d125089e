// Matrix product of 8-bit integers with a scale for each token and each output channel, on the integer
// tensor path (tcgen05.mma kind::i8, exact 32-bit sums in TMEM):
//   out[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n] + bias[n].
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace ma {
int encode_bytes_2d(CUtensorMap* out, uint64_t base, uint64_t inner, uint64_t rows, uint64_t pitch, uint32_t box_rows);

namespace {

// What gave up, as in ma_status {code, site, cta, aux}; one per device.
__device__ uint32_t g_linear_status[4];
constexpr uint32_t kCodeTimeout = 1;
constexpr uint64_t kWaitLimitNs = 2000000000ull;

__device__ __noinline__ void linear_gave_up(uint32_t site, uint32_t aux) {
  if (atomicCAS(&g_linear_status[0], 0u, kCodeTimeout) == 0u) {
    g_linear_status[1] = site;
    g_linear_status[2] = blockIdx.x;
    g_linear_status[3] = aux;
  }
}

// Bounded mbarrier wait (false: gave up).
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, uint32_t site) {
  if (mbar_test_wait(bar, parity)) return true;
  if (mbar_try_wait_for(bar, parity, 20000)) return true;
  const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
  while (!mbar_try_wait_for(bar, parity, 20000)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      linear_gave_up(site, parity);
      return false;
    }
  }
  return true;
}

// D[tmem, s32] (+)= A[smem desc, s8] * B[smem desc, s8]
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::i8: signed bytes, both operands K-major, 32-bit integer sums.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int2 ld_peer(uint32_t addr) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

struct LinearArgs {
  const float *x_scale, *w_scale;
  const uint16_t* bias;                       // (may be null)
  void* out;
  long long out_pitch;
  int tokens, inner, width, out_f32;
};

constexpr uint64_t kDescK = smem_desc_template(16, 1024);       // K-major, 128-byte swizzle
constexpr int kSlab = 128;                                      // bytes of K per stage
constexpr int kWBytes = 128 * kSlab;

// ------------------------------------------------------------------ few tokens
// The weights are the matrix instruction's 128 rows and TN tokens its columns, so that a handful of
// tokens does not run a 128-row tile of them.  One tile of 128 channels x TN tokens per cluster; its CTAs
// take a share of K each, and add their sums through each other's shared memory: integers, so the
// order does not show.
template <int TN, int STAGES>
struct Narrow {
  static constexpr int kStage = kWBytes + TN * kSlab;
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kSmem = kRing + 1024;
  static_assert(TN * 128 * 4 <= kRing, "the sums are exchanged through the ring");
};

template <int TN, int STAGES>
__global__ void __launch_bounds__(128)
linear_narrow_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                     const __grid_constant__ LinearArgs p, int splits) {
  using S = Narrow<TN, STAGES>;
  constexpr uint32_t kCols = TN < 32 ? 32 : TN;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[STAGES], s_empty[STAGES], s_done;
  __shared__ uint32_t s_tmem;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t full = smem_u32(s_full), empty = smem_u32(s_empty), done = smem_u32(&s_done);

  if (warp == 2) { tmem_alloc(smem_u32(&s_tmem), kCols); tmem_relinquish(); }
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
    mbar_init(done, 1);
    fence_mbar_init();
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  wait_for_previous();

  const int rank = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128;
  const int m0 = static_cast<int>(blockIdx.y) * TN;
  const int blocks = (p.inner + kSlab - 1) / kSlab;
  const int first = static_cast<int>(static_cast<long long>(blocks) * rank / splits);
  const int count = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / splits) - first;

  if (warp == 0) {
    if (elect_one()) {
      int sent = 0;
      for (; sent < count; ++sent) {
        const int s = sent % STAGES;
        if (sent >= STAGES && !wait_bounded(empty + 8 * s, (sent / STAGES - 1) & 1, 0x10)) break;
        const uint32_t at = ring + s * S::kStage;
        mbar_expect_tx(full + 8 * s, S::kStage);
        tma_load_2d(at, &w_map, full + 8 * s, (first + sent) * kSlab, n0);
        tma_load_2d(at + kWBytes, &x_map, full + 8 * s, (first + sent) * kSlab, m0);
      }
      if (sent < count)                       // gave up: no copy may outlive the CTA
        for (int i = sent > STAGES ? sent - STAGES : 0; i < sent; ++i)
          wait_bounded(full + 8 * (i % STAGES), (i / STAGES) & 1, 0x11);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      for (int i = 0; i < count; ++i) {
        const int s = i % STAGES;
        if (!wait_bounded(full + 8 * s, (i / STAGES) & 1, 0x12)) break;
        tc_fence_after();
        const uint32_t a = (ring + s * S::kStage) >> 4, b = a + (kWBytes >> 4);
#pragma unroll
        for (int k = 0; k < kSlab / 32; ++k)
          mma_i8(tmem, smem_desc_at(kDescK, a + 2 * k), smem_desc_at(kDescK, b + 2 * k), idesc_i8(128, TN),
                 i > 0 || k > 0);
        tc_commit(empty + 8 * s);
      }
      tc_commit(done);                        // (after a wait that gave up too: nothing is in flight then)
    }
    __syncwarp();
  }
  wait_bounded(done, 0, 0x13);
  tc_fence_after();
  __syncthreads();

  // Thread t holds channel t: its sums go to [token][channel] of this CTA's ring.
  const int valid = min(TN, p.tokens - m0);
  for (int c0 = 0; c0 < valid; c0 += 16) {
    uint32_t r[16];
    tmem_ld16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c0, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring + ((c0 + i) * 128 + tid) * 4), "r"(r[i]) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, kCols);
  if (splits > 1) { cluster_arrive(); cluster_wait(); }

  // Two channels a thread, two tokens at a time, of this CTA's share of the tokens.
  const int n = n0 + (tid & 63) * 2;
  const int t1 = static_cast<int>(static_cast<long long>(valid) * (rank + 1) / splits);
  float ws[2] = {0.f, 0.f}, bias[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (n + j < p.width) {
      ws[j] = p.w_scale[n + j];
      if (p.bias) bias[j] = __uint_as_float(static_cast<uint32_t>(p.bias[n + j]) << 16);
    }
  const int item = p.out_f32 ? 4 : 2;
  const bool pair = n + 1 < p.width && (p.out_pitch & 1) == 0 &&
                    (reinterpret_cast<uint64_t>(p.out) & (2 * item - 1)) == 0;
  for (int c = static_cast<int>(static_cast<long long>(valid) * rank / splits) + (tid >> 6); c < t1; c += 2) {
    int2 sum = make_int2(0, 0);
    const uint32_t at = ring + (c * 128 + (tid & 63) * 2) * 4;
    for (int r = 0; r < splits; ++r) {
      const int2 v = ld_peer(peer_smem(at, splits > 1 ? r : cluster_rank()));
      sum.x += v.x;
      sum.y += v.y;
    }
    const float xs = p.x_scale[m0 + c];
    const float a = static_cast<float>(sum.x) * xs * ws[0] + bias[0];
    const float b = static_cast<float>(sum.y) * xs * ws[1] + bias[1];
    const long long o = static_cast<long long>(m0 + c) * p.out_pitch + n;
    if (p.out_f32) {
      float* out = static_cast<float*>(p.out) + o;
      if (pair) *reinterpret_cast<float2*>(out) = make_float2(a, b);
      else {
        if (n < p.width) out[0] = a;
        if (n + 1 < p.width) out[1] = b;
      }
    } else {
      uint16_t* out = static_cast<uint16_t*>(p.out) + o;
      const uint32_t v = pack_bf16x2(a, b);
      if (pair) *reinterpret_cast<uint32_t*>(out) = v;
      else {
        if (n < p.width) out[0] = static_cast<uint16_t>(v);
        if (n + 1 < p.width) out[1] = static_cast<uint16_t>(v >> 16);
      }
    }
  }
  if (splits > 1) { cluster_arrive(); cluster_wait(); }     // (peers read this CTA's sums until here)
}

template <int TN, int STAGES>
cudaError_t launch_narrow(const CUtensorMap& w, const CUtensorMap& x, const LinearArgs& p, int splits,
                          cudaStream_t stream) {
  using S = Narrow<TN, STAGES>;
  auto kernel = linear_narrow_kernel<TN, STAGES>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.width + 127) / 128 * splits), static_cast<unsigned>((p.tokens + TN - 1) / TN));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, w, x, p, splits);
  const cudaError_t last = cudaGetLastError();
  return e != cudaSuccess ? e : last;
}

}  // namespace
}  // namespace ma

extern "C" int ma_linear_quant(const ma_linear_quant_args* a, void* stream_) {
  if (!a || !a->x || !a->weight || !a->x_scale || !a->weight_scale || !a->out) return MA_ERR_INVALID;
  if (a->tokens < 0 || a->width < 0 || a->inner < 1) return MA_ERR_INVALID;
  if (a->inner > 131071 || a->tokens > (1 << 30) || a->width > (1 << 30)) return MA_ERR_CAPACITY;
  if ((a->x & 15u) || (a->weight & 15u) || (a->x_pitch & 15) || (a->weight_pitch & 15) || a->x_pitch < a->inner ||
      a->weight_pitch < a->inner || a->out_pitch < a->width)
    return MA_ERR_INVALID;
  if ((a->x_scale & 3u) || (a->weight_scale & 3u) || (a->bias & 1u) || (a->out & (a->out_f32 ? 3u : 1u)))
    return MA_ERR_INVALID;
  if (a->tokens == 0 || a->width == 0) return MA_OK;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return MA_ERR_CUDA;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  ma::LinearArgs p{};
  p.x_scale = reinterpret_cast<const float*>(a->x_scale);
  p.w_scale = reinterpret_cast<const float*>(a->weight_scale);
  p.bias = reinterpret_cast<const uint16_t*>(a->bias);
  p.out = reinterpret_cast<void*>(a->out);
  p.out_pitch = a->out_pitch;
  p.tokens = a->tokens; p.inner = a->inner; p.width = a->width; p.out_f32 = a->out_f32;
  const int tn = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : p.tokens <= 128 ? 128 : 256;
  const long long rows = (p.tokens + tn - 1) / tn;
  if (rows > 65535) return MA_ERR_CAPACITY;
  const long long tiles = (p.width + 127) / 128 * rows;
  const int blocks = (p.inner + 127) / 128;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 2 * sms && blocks >= splits * 4) splits *= 2;
  CUtensorMap w, x;
  int rc = ma::encode_bytes_2d(&w, a->weight, static_cast<uint64_t>(p.inner), static_cast<uint64_t>(p.width),
                               static_cast<uint64_t>(a->weight_pitch), 128);
  if (rc == MA_OK)
    rc = ma::encode_bytes_2d(&x, a->x, static_cast<uint64_t>(p.inner), static_cast<uint64_t>(p.tokens),
                             static_cast<uint64_t>(a->x_pitch), static_cast<uint32_t>(tn));
  if (rc != MA_OK) return rc;
  cudaError_t e;
  switch (tn) {
    case 16: e = ma::launch_narrow<16, 6>(w, x, p, splits, stream); break;
    case 32: e = ma::launch_narrow<32, 5>(w, x, p, splits, stream); break;
    case 64: e = ma::launch_narrow<64, 4>(w, x, p, splits, stream); break;
    case 128: e = ma::launch_narrow<128, 3>(w, x, p, splits, stream); break;
    default: e = ma::launch_narrow<256, 4>(w, x, p, splits, stream); break;
  }
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

extern "C" int ma_linear_status(void* stream, ma_status* out) {
  if (!out) return MA_ERR_INVALID;
  uint32_t h[4] = {0, 0, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaMemcpyFromSymbolAsync(h, ma::g_linear_status, sizeof(h), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return MA_ERR_CUDA;
  out->code = h[0]; out->site = h[1]; out->cta = h[2]; out->aux = h[3];
  if (h[0] == 0) return MA_OK;
  const uint32_t zero[4] = {0, 0, 0, 0};
  if (cudaMemcpyToSymbolAsync(ma::g_linear_status, zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return MA_ERR_CUDA;
  return MA_ERR_DEVICE_TIMEOUT;
}
