// Matrix product of 8-bit integers with a scale for each token and each output channel, on the integer
// tensor path (tcgen05.mma kind::i8, exact 32-bit sums in TMEM):
//   out[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n] + bias[n].
// The sum is converted to fp32, scaled and biased there, and rounded once to the output's type.
//
// With few tokens the weights' way from memory bounds it (one byte per weight), with many the tensor cores
// (8192 products per cycle and SM) and, in a long run, the power limit.  Two kernels, each in a few widths;
// linear_form.h says which and why.  Device time in a chain of calls, inputs from memory:
//   tokens x inner x width       time      of the measured copy rate / of twice the measured bf16 rate
//       1 x  4096 x 10240      8.9 us      0.73 of the copy rate
//      48 x 16384 x  2304     10.8 us      0.56
//    1384 x  4096 x  1280     10.1 us      0.43 of the burst rate (3365 TOP/s)
//   13400 x  4096 x 10240      351 us      0.95; back to back for a second 412 us, 0.98 of the sustained (2781)
//   22600 x  4096 x 16384      937 us      0.96; 1102 us, 0.99
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "../../include/megaattn_b200.h"
#include "launch.cuh"
#include "linear_form.h"
#include "ptx.cuh"

namespace ma {
int encode_bytes_2d(CUtensorMap* out, uint64_t base, uint64_t inner, uint64_t rows, uint64_t pitch, uint32_t box_rows);
int encode_out_2d(CUtensorMap* out, uint64_t base, bool f32, uint64_t cols, uint64_t rows, uint64_t pitch_bytes,
                  uint32_t box_bytes);

namespace {

// What gave up first since the last report, in one word that is taken and cleared in one step: code, site and aux of
// a byte each (of ma_status), and the CTA.  One per device, so a report takes what any stream's calls left.
__device__ unsigned long long g_linear_status, g_linear_taken;
constexpr uint32_t kCodeTimeout = 1;
// What a CTA that gave up passes on instead of its sums: no sum of 131071 products of bytes is that low.  The
// outputs that depend on it are NaN, as are those of the tiles that a pair which gave up did not get to.
constexpr int kNoSum = static_cast<int>(0x80000000u);
constexpr uint32_t kNaN = 0x7fc00000u;
// A call waits for its own copies and products only, never for another kernel or GPU: no argument sets this.
#ifdef MA_AUDIT
constexpr uint64_t kWaitLimitNs = 200000000ull;
// {copies of a CTA that gave up that it had not seen land, those of them that it waited for, CTAs that gave up}
__device__ uint32_t g_linear_audit[3];
#else
constexpr uint64_t kWaitLimitNs = 2000000000ull;
#endif

__device__ __noinline__ void linear_gave_up(uint32_t site, uint32_t aux) {
  atomicCAS(&g_linear_status, 0ull,
            kCodeTimeout | (site & 255u) << 8 | (aux & 255u) << 16 | static_cast<unsigned long long>(blockIdx.x) << 32);
}
__global__ void linear_take_status() { g_linear_taken = atomicExch(&g_linear_status, 0ull); }

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

// For a CTA that gave up: the last copy into each of `stages` stages, the first `turn` of which are a lap ahead of the
// others (`parity` is theirs).
__device__ __noinline__ void wait_for_copies(uint32_t full, int stages, int turn, uint32_t parity, uint32_t site) {
  for (int i = 0; i < stages; ++i) {
    const bool landed = wait_bounded(full + 8 * i, i < turn ? parity : parity ^ 1u, site);
#ifdef MA_AUDIT
    atomicAdd(&g_linear_audit[0], 1u);
    atomicAdd(&g_linear_audit[1], landed ? 1u : 0u);
    if (i == 0) atomicAdd(&g_linear_audit[2], 1u);
#endif
    (void)landed;
  }
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
// The same for what needs no order of memory: that a CTA's shared memory lives on, or barriers that a fence of
// their own has published.  (With release it waits for the thread's stores: 1500 to 2500 cycles at the end.)
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
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
__device__ __forceinline__ int4 ld_peer(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Brings a box to L2 only: no value is read, so it may run before what precedes the launch is complete.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}

struct LinearArgs {
  const float *x_scale, *w_scale;
  const uint16_t* bias;                       // (may be null)
  void* out;
  long long out_pitch;
  int tokens, inner, width, out_f32;
#ifdef MA_AUDIT
  int stall;                                  // block of K at which the issuer waits for what nobody sends (-1: none)
#endif
};

constexpr uint64_t kDescK = smem_desc_template(16, 1024);       // K-major, 128-byte swizzle
constexpr int kSlab = kLinearSlab;
constexpr int kWBytes = 128 * kSlab;

// ------------------------------------------------------------------ few tokens
// The weights are the matrix instruction's 128 rows and TN tokens its columns, so that a handful of
// tokens does not run a 128-row tile of them.  One tile of 128 channels x TN tokens per cluster; its CTAs
// take a share of K each, and add their sums through each other's shared memory: integers, so the
// order does not show.  Every CTA has 64 to 180 KB on their way; what is left beside the loads is the start
// of a kernel and of its first load, the exchange, and the end (1 x 512 x 512 takes 2.7 us).
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

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
  __shared__ uint32_t s_tmem, s_gave_up, s_sent;
  __shared__ float s_xs[TN];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t full = smem_u32(s_full), empty = smem_u32(s_empty), done = smem_u32(&s_done);

  if (warp == 2) { tmem_alloc(smem_u32(&s_tmem), kCols); tmem_relinquish(); }
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
    mbar_init(done, 1);
    s_gave_up = 0;
    fence_mbar_init();
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  let_next_start();

  const int rank = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128;
  const int m0 = static_cast<int>(blockIdx.y) * TN;
  const int blocks = (p.inner + kSlab - 1) / kSlab;
  const int first = static_cast<int>(static_cast<long long>(blocks) * rank / splits);
  const int count = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / splits) - first;
  if (tid == 0)                               // the weights are on their way while the kernel before ends
    for (int i = 0; i < min(count, STAGES); ++i) tma_prefetch_2d(&w_map, (first + i) * kSlab, n0);
  wait_for_previous();

  if (warp == 0) {
    if (elect_one()) {
      int sent = 0;
      for (; sent < count; ++sent) {
        const int s = sent % STAGES;
        if (sent >= STAGES && !wait_bounded(empty + 8 * s, (sent / STAGES - 1) & 1, 0x10)) { s_gave_up = 1; break; }
        const uint32_t at = ring + s * S::kStage;
        mbar_expect_tx(full + 8 * s, S::kStage);
        tma_load_2d(at, &w_map, full + 8 * s, (first + sent) * kSlab, n0);
        tma_load_2d(at + kWBytes, &x_map, full + 8 * s, (first + sent) * kSlab, m0);
      }
      s_sent = static_cast<uint32_t>(sent);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      for (int i = 0; i < count; ++i) {
        const int s = i % STAGES;
        uint32_t bar = full + 8 * s, parity = (i / STAGES) & 1;
#ifdef MA_AUDIT
        if (first + i == p.stall) { bar = done; parity = 0; }
#endif
        if (!wait_bounded(bar, parity, 0x12)) { s_gave_up = 1; break; }
        tc_fence_after();
        const uint32_t a = (ring + s * S::kStage) >> 4, b = a + (kWBytes >> 4);
#pragma unroll
        for (int k = 0; k < kSlab / 32; ++k)
          mma_i8(tmem, smem_desc_at(kDescK, a + 2 * k), smem_desc_at(kDescK, b + 2 * k), idesc_i8(128, TN),
                 i > 0 || k > 0);
        tc_commit(empty + 8 * s);
      }
      tc_commit(done);                        // (after a wait that gave up too)
    }
    __syncwarp();
  }
  // Four channels a lane in the end; their scales and the tokens' are fetched under the loads.
  const int lane = tid & 31, valid = min(TN, p.tokens - m0), n = n0 + lane * 4;
  float ws[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ws[j] = n + j < p.width ? p.w_scale[n + j] : 0.f;
    bias[j] = p.bias && n + j < p.width ? __uint_as_float(static_cast<uint32_t>(p.bias[n + j]) << 16) : 0.f;
  }
  for (int c = tid; c < valid; c += 128) s_xs[c] = p.x_scale[m0 + c];
  if (!wait_bounded(done, 0, 0x13)) s_gave_up = 1;
  tc_fence_after();
  __syncthreads();
  if (s_gave_up) {
    // Whichever wait it was: no copy may land in what is the sums' from here on, or outlive the CTA.  Where the
    // issuer gave up the producer has sent on, so every stage's last copy is waited for.
    if (tid == 0) wait_for_copies(full, STAGES, static_cast<int>(s_sent % STAGES), s_sent / STAGES & 1u, 0x11);
    __syncthreads();
  }

  // Thread t holds channel t: its sums go to [token][channel] of this CTA's ring.
  if (s_gave_up) {
#pragma unroll 1
    for (int i = 0; i < TN; ++i)
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring + (i * 128 + tid) * 4), "r"(kNoSum) : "memory");
  } else {
    constexpr int kCol = TN < 32 ? 16 : 32;
    uint32_t r[TN / kCol][kCol];
#pragma unroll
    for (int i = 0; i < TN / kCol; ++i) tmem_ld_columns(tmem + (static_cast<uint32_t>(warp * 32) << 16) + i * kCol, r[i]);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < TN; ++i)
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring + (i * 128 + tid) * 4), "r"(r[i / kCol][i % kCol]) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, kCols);
  if (splits > 1) { cluster_arrive(); cluster_wait(); }

  // Every CTA adds up its share of the tokens, a warp two at a time, all parts of both in flight.
  const int t1 = valid * (rank + 1) / splits;
  const int item = p.out_f32 ? 4 : 2;
  const bool whole = n + 4 <= p.width && ((reinterpret_cast<uint64_t>(p.out) | static_cast<uint64_t>(p.out_pitch) * item) &
                                          (4u * item - 1)) == 0;
  const uint32_t mine = splits > 1 ? 0 : cluster_rank();
  for (int c = valid * rank / splits + warp; c < t1; c += 8) {
    int4 part[2][kMaxSplits];
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      const uint32_t at = peer_smem(ring + (c * 128 + lane * 4) * 4, mine + (r < splits ? r : 0));
#pragma unroll
      for (int u = 0; u < 2; ++u)
        part[u][r] = r < splits && c + 4 * u < t1 ? ld_peer(at + u * 2048) : make_int4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (c + 4 * u >= t1) break;
      int sum[4] = {0, 0, 0, 0};
      bool lost = false;
#pragma unroll
      for (int r = 0; r < kMaxSplits; ++r) {
        lost |= part[u][r].x == kNoSum;
        sum[0] += part[u][r].x;
        sum[1] += part[u][r].y;
        sum[2] += part[u][r].z;
        sum[3] += part[u][r].w;
      }
      const float xs = lost ? __uint_as_float(kNaN) : s_xs[c + 4 * u];
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(static_cast<float>(sum[j]) * xs, ws[j], bias[j]);
      const long long o = static_cast<long long>(m0 + c + 4 * u) * p.out_pitch + n;
      if (p.out_f32) {
        float* out = static_cast<float*>(p.out) + o;
        if (whole) {
          *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.width) out[j] = v[j];
        }
      } else {
        uint16_t* out = static_cast<uint16_t*>(p.out) + o;
        const uint2 w = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        if (whole) {
          *reinterpret_cast<uint2*>(out) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.width) out[j] = static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
        }
      }
    }
  }
  // Peers read this CTA's sums until here.  Relaxed is enough on their side too: what a warp has loaded from them is in
  // its registers by now, as its stores above were made of it, and those are no business of the peers.
  if (splits > 1) { cluster_arrive_relaxed(); cluster_wait(); }
}

// A kernel's shared memory beyond 48 KB, allowed once per device (an attribute that outlasts the call; to
// set it twice does no harm).
template <class K>
cudaError_t allow_smem(K kernel, int bytes, int dev, std::atomic<uint64_t>* done) {
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

#ifdef MA_AUDIT
int g_linear_stall = -1;
#endif

// The tensor maps and the launch; an ma_error.
template <int TN, int STAGES>
int launch_narrow(const ma_linear_quant_args* a, const LinearArgs& p, int splits, int dev, cudaStream_t stream) {
  using S = Narrow<TN, STAGES>;
  CUtensorMap w, x;
  const uint64_t inner = static_cast<uint64_t>(p.inner);
  int rc = encode_bytes_2d(&w, a->weight, inner, static_cast<uint64_t>(p.width), static_cast<uint64_t>(a->weight_pitch),
                           128);
  if (rc == MA_OK)
    rc = encode_bytes_2d(&x, a->x, inner, static_cast<uint64_t>(p.tokens), static_cast<uint64_t>(a->x_pitch), TN);
  if (rc != MA_OK) return rc;
  auto kernel = linear_narrow_kernel<TN, STAGES>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(kernel, S::kSmem, dev, &allowed);
  if (e != cudaSuccess) return MA_ERR_CUDA;
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
  return e == cudaSuccess && last == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

// ------------------------------------------------------------------ many tokens
// Two SMs share a tile of 256 tokens x BN channels (cta_group::2): each brings 128 token rows and half of
// the weight rows, and one issuer runs both tensor cores, so a byte of either operand is loaded once per
// pair.  Persistent pairs walk the tiles, 8 tiles of tokens at a time so that what runs at once shares its
// operands in L2; the sums are double-buffered in TMEM, so the epilogue of a tile runs under the next.
// An SM takes in 64 bytes a cycle at most, which is what a tile of 256 channels asks for (32 KB per 512 cycles
// of products); tiles of 512, single-buffered in two halves, ask for 48 and were slower (4096 x 4096 x 4096
// 50 us for 48) until K is 16384 long (208 for 218).  4096 x 4096 x 4096: tensor cores 81 % busy, 48 us.
template <int BN, int STAGES, bool F32>
struct Wide {
  static constexpr int kA = 128 * kSlab, kB = BN / 2 * kSlab, kStage = kA + kB;
  static constexpr int kRow = !F32 && BN == 64 ? 64 : 128;      // bytes of a staged row
  static constexpr int kStaging = STAGES * kStage;              // 8 warps x 32 rows
  static constexpr int kCols = kStaging + 8 * 4096;             // 2 x {scale, bias} x BN
  static constexpr int kSmem = kCols + 2 * 2 * BN * 4 + 1024;
};
constexpr int kWideThreads = 384;            // producer, issuer, TMEM, (idle), 8 warps for the epilogue

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this address in both CTAs once every MMA issued so far completed.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
// A load into this CTA's shared memory that is counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// An arrival on a barrier of either CTA, for what tcgen05 fences order.  (With release semantics at cluster
// scope it waited for the thread's stores, 1200 to 2700 cycles of a tile's epilogue.)
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __noinline__ void fill_nan(void* out, bool f32, long long row, int n, int end) {
  for (; n < end; ++n) {
    if (f32) static_cast<uint32_t*>(out)[row + n] = kNaN;
    else static_cast<uint16_t*>(out)[row + n] = static_cast<uint16_t>(kNaN >> 16);
  }
}

struct WideTiles {
  int m, n, total, stored;                   // stored: the output takes TMA stores (16-byte rows)
};
constexpr int kGroupM = 8;                   // tiles of tokens that are walked together
__device__ __forceinline__ void tile_at(const WideTiles& t, int i, int* m, int* n) {
  const int per = kGroupM * t.n, g = i / per, r = i - g * per;
  const int gm = min(kGroupM, t.m - g * kGroupM);
  *n = r / gm;
  *m = g * kGroupM + r - *n * gm;
}

// 32 sums of a row to 32 outputs, two at a time.
template <bool BIASED>
__device__ __forceinline__ void scale_columns(const uint32_t (&r)[32], uint64_t xs, uint32_t cols, uint32_t bias_at,
                                              float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 s = ld_shared_f32x4(cols + j * 4);
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (BIASED) b = ld_shared_f32x4(cols + bias_at + j * 4);
    const uint64_t lo = mul_f32x2(pack_f32x2(static_cast<float>(static_cast<int>(r[j])),
                                             static_cast<float>(static_cast<int>(r[j + 1]))), xs);
    const uint64_t hi = mul_f32x2(pack_f32x2(static_cast<float>(static_cast<int>(r[j + 2])),
                                             static_cast<float>(static_cast<int>(r[j + 3]))), xs);
    unpack_f32x2(fma_f32x2(lo, pack_f32x2(s.x, s.y), pack_f32x2(b.x, b.y)), v[j], v[j + 1]);
    unpack_f32x2(fma_f32x2(hi, pack_f32x2(s.z, s.w), pack_f32x2(b.z, b.w)), v[j + 2], v[j + 3]);
  }
}
// This lane's row into the warp's staging: ROW bytes, 16-byte pieces swizzled as the output's tensor map has it.
template <int ROW>
__device__ __forceinline__ void put_row(const uint32_t* u, uint32_t staging, int lane) {
  const uint32_t flip = ROW == 128 ? lane & 7 : (lane >> 1) & 3;
#pragma unroll
  for (int j = 0; j < ROW / 16; ++j)
    st_shared_v4(staging + lane * ROW + ((j ^ flip) << 4), u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
}
// Staged rows to rows that do not start at 16 bytes, and a row's last columns (TMA writes 16 bytes at a time,
// beyond the last column too): 16 bytes at a time where the output has them, ROW / 16 lanes a row, and what is
// left on either side by elements.  `bytes` of each of `rows` rows.  A batch is read before any of it is
// written: one at a time, every row waited for its words.
template <int ITEM, int ROW>
__device__ __forceinline__ void copy_rows(uint32_t staging, char* out, long long pitch, int rows, int bytes, int lane) {
  constexpr int kPieces = ROW / 16, kRows = 32 / kPieces, kBatch = 4;
  auto piece = [&](int row, int j) {         // where a staged row's j-th 16 bytes are
    return staging + row * ROW + (((j & (kPieces - 1)) ^ (ROW == 128 ? row & 7 : (row >> 1) & 3)) << 4);
  };
  {
    const int j = lane % kPieces;
    const long long step = pitch * kRows;
    char* to = out + lane / kPieces * pitch;
#pragma unroll 1
    for (int r0 = lane / kPieces; r0 < rows; r0 += kBatch * kRows, to += kBatch * step) {
      uint32_t w[kBatch][8];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {     // (row 31 and below, whatever `rows` is)
        const int r = (r0 + i * kRows) & 31;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[i][4 * h]), "=r"(w[i][4 * h + 1]), "=r"(w[i][4 * h + 2]), "=r"(w[i][4 * h + 3])
                       : "r"(piece(r, j + h)));
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        char* row = to + i * step;
        const int head = -static_cast<int>(reinterpret_cast<uint64_t>(row)) & 15;
        uint32_t* x = w[i];
        if (head & 8) {
#pragma unroll
          for (int k = 0; k < 6; ++k) x[k] = x[k + 2];
        }
        if (head & 4) {
#pragma unroll
          for (int k = 0; k < 5; ++k) x[k] = x[k + 1];
        }
        if (ITEM == 2 && (head & 2)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = __funnelshift_r(x[k], x[k + 1], 16);
        }
        if (r0 + i * kRows < rows && head + j * 16 + 16 <= bytes)
          *reinterpret_cast<uint4*>(row + head + j * 16) = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  }
  constexpr int kSide = 16 / ITEM, kSideRows = 32 / (2 * kSide), kSides = 8;
  const int e = lane % kSide * ITEM;
  const bool left = lane % (2 * kSide) < kSide;
  const long long step = pitch * kSideRows;
  char* to = out + lane / (2 * kSide) * pitch;
#pragma unroll 1
  for (int r0 = lane / (2 * kSide); r0 < rows; r0 += kSides * kSideRows, to += kSides * step) {
    uint32_t w[kSides];
    int at[kSides];
#pragma unroll
    for (int i = 0; i < kSides; ++i) {
      const int head = min(-static_cast<int>(reinterpret_cast<uint64_t>(to + i * step)) & 15, bytes);
      at[i] = left ? e : head + ((bytes - head) & ~15) + e;
      const uint32_t from = piece((r0 + i * kSideRows) & 31, at[i] >> 4) + (at[i] & 15);
      if (ITEM == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(from));
      else asm volatile("{\n\t.reg .u16 t;\n\tld.shared.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(w[i]) : "r"(from));
      if (r0 + i * kSideRows >= rows || at[i] >= (left ? head : bytes)) at[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < kSides; ++i) {
      if (at[i] < 0) continue;
      if (ITEM == 4) *reinterpret_cast<uint32_t*>(to + i * step + at[i]) = w[i];
      else *reinterpret_cast<uint16_t*>(to + i * step + at[i]) = static_cast<uint16_t>(w[i]);
    }
  }
}

template <int BN, int STAGES, bool F32>
__global__ void __launch_bounds__(kWideThreads)
linear_wide_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                   const __grid_constant__ CUtensorMap out_map, const __grid_constant__ LinearArgs p,
                   const WideTiles tiles) {
  using S = Wide<BN, STAGES, F32>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[STAGES], s_empty[STAGES], s_acc_full[2], s_acc_empty[2];
  __shared__ uint32_t s_tmem;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full = smem_u32(s_full), empty = smem_u32(s_empty);
  const uint32_t acc_full = smem_u32(s_acc_full), acc_empty = smem_u32(s_acc_empty);
  const uint32_t rank = cluster_rank();

  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&s_tmem)), "r"(2 * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, 16); }
    fence_mbar_init();
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
    if (tiles.stored) tma_prefetch_desc(&out_map);
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_relaxed();                  // (the other CTA's barriers are set up)
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  let_next_start();

  const int blocks = (p.inner + kSlab - 1) / kSlab;
  const int pair = static_cast<int>(blockIdx.x) >> 1, pairs = static_cast<int>(gridDim.x) >> 1;
  if (threadIdx.x == 0) {                    // the weights are on their way while the kernel before ends
    int tm, tn;
    tile_at(tiles, pair, &tm, &tn);
    for (int k = 0; k < min(blocks, STAGES); ++k)
      tma_prefetch_2d(&w_map, k * kSlab, tn * BN + static_cast<int>(rank) * (BN / 2));
  }
  wait_for_previous();

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, phase = 0;
      bool ok = true;
      for (int i = pair; i < tiles.total && ok; i += pairs) {
        int tm, tn;
        tile_at(tiles, i, &tm, &tn);
        const int m0 = tm * 256 + static_cast<int>(rank) * 128, n0 = tn * BN + static_cast<int>(rank) * (BN / 2);
        for (int k = 0; k < blocks; ++k) {
          ok = wait_bounded(empty + 8 * s, phase ^ 1u, 0x20);
          if (!ok) break;
          if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * S::kStage);
          const uint32_t at = ring + s * S::kStage, bar = peer_smem(full + 8 * s, 0);
          tma_load_2d_pair(at, &x_map, bar, k * kSlab, m0);
          tma_load_2d_pair(at + S::kA, &w_map, bar, k * kSlab, n0);
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
      }
      // every load is used, and no arrival on a barrier of this CTA outstanding, before it ends
      const uint32_t end = s, end_phase = phase;
      for (int i = 0; i < STAGES && ok; ++i) {
        ok = wait_bounded(empty + 8 * s, phase ^ 1u, 0x24);
        if (++s == STAGES) { s = 0; phase ^= 1u; }
      }
      // Gave up: no copy may outlive the pair.  Those of both CTAs are counted here, and the other one waits at
      // the end of the kernel; a stage's last load was in this phase before `end`, in the one before from there on.
      if (!ok && rank == 0) wait_for_copies(full, STAGES, static_cast<int>(end), end_phase, 0x25);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      uint32_t s = 0, phase = 0, it = 0;
      bool ok = true;
      for (int i = pair; i < tiles.total && ok; i += pairs, ++it) {
        const uint32_t acc = it & 1u, d = tmem + acc * BN;
        ok = wait_bounded(acc_empty + 8 * acc, ((it >> 1) & 1u) ^ 1u, 0x21);
        tc_fence_after();
        for (int k = 0; k < blocks && ok; ++k) {
          uint32_t bar = full + 8 * s, parity = phase;
#ifdef MA_AUDIT
          if (it == 0 && k == p.stall) { bar = acc_full; parity = 0; }
#endif
          ok = wait_bounded(bar, parity, 0x22);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = (ring + s * S::kStage) >> 4, b = a + (S::kA >> 4);
#pragma unroll
          for (int j = 0; j < kSlab / 32; ++j)
            mma_i8_pair(d, smem_desc_at(kDescK, a + 2 * j), smem_desc_at(kDescK, b + 2 * j), idesc_i8(256, BN),
                        k > 0 || j > 0);
          tc_commit_pair(empty + 8 * s);
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
        if (ok) tc_commit_pair(acc_full + 8 * acc);      // (a tile that is not complete is not passed on)
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // Warps 4-7 take the first half of the columns, 8-11 the second; a warp reads the TMEM lanes of its
    // number mod 4.  They meet at a barrier per tile, so a warp whose wait gave up goes through the
    // remaining tiles without work rather than leave.
    const int w = warp - 4, first = (w >> 2) * (BN / 2), e = threadIdx.x - 128;
    const uint32_t staging = ring + S::kStaging + w * 4096;
    constexpr int kItem = F32 ? 4 : 2, kChunk = S::kRow / kItem;      // columns of a staged row
    uint32_t it = 0;
    bool ok = true;
    for (int i = pair; i < tiles.total; i += pairs, ++it) {
      const uint32_t acc = it & 1u;
      int tm, tn;
      tile_at(tiles, i, &tm, &tn);
      const int row0 = tm * 256 + static_cast<int>(rank) * 128 + (w & 3) * 32, n0 = tn * BN;
      const int rows = min(32, p.tokens - row0);             // (none or less: beyond the last token)
      const float xs = lane < rows ? p.x_scale[row0 + lane] : 0.f;
      const uint64_t xs2 = pack_f32x2(xs, xs);
      const uint32_t cols = ring + S::kCols + acc * (2 * BN * 4);
      if (e < BN) {
        const int n = n0 + e;
        st_shared_f32(cols + e * 4, n < p.width ? p.w_scale[n] : 0.f);
        if (p.bias)
          st_shared_f32(cols + (BN + e) * 4,
                        n < p.width ? __uint_as_float(static_cast<uint32_t>(p.bias[n]) << 16) : 0.f);
      }
      named_bar_sync(1, kWideThreads - 128);
      if (ok) ok = wait_bounded(acc_full + 8 * acc, (it >> 1) & 1u, 0x23);
      if (!ok) {
        if (lane < rows) fill_nan(p.out, F32, static_cast<long long>(row0 + lane) * p.out_pitch, n0 + first, min(n0 + first + BN / 2, p.width));
        continue;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + acc * BN + first + (static_cast<uint32_t>((w & 3) * 32) << 16);
      uint32_t r[2][32], u[S::kRow / 4];       // (u: a staged row)
      tmem_ld32(taddr, r[0]);
#pragma unroll
      for (int c = 0; c < BN / 64; ++c) {
        tc_wait_ld();
        if (c + 1 < BN / 64) {
          tmem_ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
        } else {                             // all of this warp's sums are out of TMEM
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_peer(peer_smem(acc_empty + 8 * acc, 0));
        }
        const int n = n0 + first + c * 32, chunk = n / kChunk * kChunk;
        if (rows <= 0 || chunk >= p.width) continue;                   // (the same for the warp)
        float v[32];
        if (p.bias) scale_columns<true>(r[c & 1], xs2, cols + (first + c * 32) * 4, BN * 4, v);
        else scale_columns<false>(r[c & 1], xs2, cols + (first + c * 32) * 4, BN * 4, v);
        constexpr int kWords = F32 ? 32 : 16;          // of 32 columns
#pragma unroll
        for (int j = 0; j < kWords; ++j)
          u[c * kWords % (S::kRow / 4) + j] = F32 ? __float_as_uint(v[j]) : pack_bf16x2(v[2 * j % 32], v[(2 * j + 1) % 32]);
        if (n + 32 < chunk + kChunk) continue;
        // (the staging is written as late as can be: the store before has to have read it)
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
        put_row<S::kRow>(u, staging, lane);
        if (tiles.stored && chunk + kChunk <= p.width) {     // TMA leaves out rows beyond the last
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&out_map, staging, chunk, row0);
            tma_store_commit();
          }
        } else {
          __syncwarp();
          copy_rows<kItem, S::kRow>(staging,
                                    static_cast<char*>(p.out) + (static_cast<long long>(row0) * p.out_pitch + chunk) * kItem,
                                    p.out_pitch * kItem, rows, min(kChunk, p.width - chunk) * kItem, lane);
          __syncwarp();
        }
      }
    }
    if (lane == 0) tma_store_wait_read();    // (the staging lives until its last store has read it)
    __syncwarp();
  }
  __syncthreads();
  tc_fence_before();
  cluster_arrive_relaxed();                  // (barriers and sums of a CTA are used by the other)
  cluster_wait();
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
}

template <int BN, int STAGES, bool F32>
cudaError_t launch_wide_as(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& out, bool stored,
                           const LinearArgs& p, int sms, int dev, cudaStream_t stream) {
  using S = Wide<BN, STAGES, F32>;
  static_assert(S::kSmem + 256 <= 232448, "shared memory of an SM");
  auto kernel = linear_wide_kernel<BN, STAGES, F32>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(kernel, S::kSmem, dev, &allowed);
  if (e != cudaSuccess) return e;
  WideTiles t;
  t.m = (p.tokens + 255) / 256;
  t.n = (p.width + BN - 1) / BN;
  t.total = t.m * t.n;
  t.stored = stored;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (t.total < sms / 2 ? t.total : sms / 2)));
  cfg.blockDim = dim3(kWideThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, w, x, out, p, t);
  const cudaError_t last = cudaGetLastError();
  return e != cudaSuccess ? e : last;
}

// The tensor maps and the launch; an ma_error.
template <int BN, int STAGES>
int launch_wide(const ma_linear_quant_args* a, const LinearArgs& p, int sms, int dev, cudaStream_t stream) {
  CUtensorMap w, x, out{};
  const uint64_t inner = static_cast<uint64_t>(p.inner), pitch = static_cast<uint64_t>(p.out_pitch) * (p.out_f32 ? 4 : 2);
  const bool stored = ((a->out | pitch) & 15u) == 0;
  int rc = encode_bytes_2d(&w, a->weight, inner, static_cast<uint64_t>(p.width), static_cast<uint64_t>(a->weight_pitch),
                           BN / 2);
  if (rc == MA_OK)
    rc = encode_bytes_2d(&x, a->x, inner, static_cast<uint64_t>(p.tokens), static_cast<uint64_t>(a->x_pitch), 128);
  if (rc == MA_OK && stored)
    rc = encode_out_2d(&out, a->out, p.out_f32 != 0, static_cast<uint64_t>(p.width), static_cast<uint64_t>(p.tokens),
                       pitch, p.out_f32 ? Wide<BN, STAGES, true>::kRow : Wide<BN, STAGES, false>::kRow);
  if (rc != MA_OK) return rc;
  const cudaError_t e = p.out_f32 ? launch_wide_as<BN, STAGES, true>(w, x, out, stored, p, sms, dev, stream)
                                  : launch_wide_as<BN, STAGES, false>(w, x, out, stored, p, sms, dev, stream);
  return e == cudaSuccess ? MA_OK : MA_ERR_CUDA;
}

int linear_dispatch(const ma_linear_quant_args* a, const LinearArgs& p, int sms, int dev, cudaStream_t stream) {
  const LinearForm f = linear_form(p.tokens, p.inner, p.width, sms);
  // (tiles are counted in 32 bits, a round beyond the last)
  if (f.tiles > (f.splits ? 0x7fffffffLL : 0x7fff0000LL)) return MA_ERR_CAPACITY;
  switch (f.splits ? f.stages : 0) {
    case 11: return launch_narrow<16, 11>(a, p, f.splits, dev, stream);
    case 6: return launch_narrow<16, 6>(a, p, f.splits, dev, stream);
    case 10: return launch_narrow<32, 10>(a, p, f.splits, dev, stream);
    case 5: return launch_narrow<32, 5>(a, p, f.splits, dev, stream);
    case 8: return launch_narrow<64, 8>(a, p, f.splits, dev, stream);
    case 4: return launch_narrow<64, 4>(a, p, f.splits, dev, stream);
    default: break;
  }
  switch (f.width) {
    case 64: return launch_wide<64, 9>(a, p, sms, dev, stream);
    case 128: return launch_wide<128, 7>(a, p, sms, dev, stream);
    default: return launch_wide<256, 5>(a, p, sms, dev, stream);
  }
}

}  // namespace
}  // namespace ma

#ifdef MA_AUDIT
// Test build: the following calls' issuers wait for what nobody sends at this block of K (-1: they do not).
extern "C" void ma_audit_linear_stall(int block) { ma::g_linear_stall = block; }
// g_linear_audit since the last call, which it clears.
extern "C" int ma_audit_linear_counts(uint32_t* out) {
  const uint32_t zero[3] = {0, 0, 0};
  return cudaMemcpyFromSymbol(out, ma::g_linear_audit, sizeof(zero)) == cudaSuccess &&
                 cudaMemcpyToSymbol(ma::g_linear_audit, zero, sizeof(zero)) == cudaSuccess
             ? MA_OK : MA_ERR_CUDA;
}
#endif

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
#ifdef MA_AUDIT
  p.stall = ma::g_linear_stall;
#endif
  return ma::linear_dispatch(a, p, sms, dev, stream);
}

extern "C" int ma_linear_status(void* stream, ma_status* out) {
  if (!out) return MA_ERR_INVALID;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaStreamSynchronize(s) != cudaSuccess) return MA_ERR_CUDA;
  static std::mutex one_at_a_time;             // (g_linear_taken is every report's; the long wait is over)
  const std::lock_guard<std::mutex> lock(one_at_a_time);
  unsigned long long w = 0;
  ma::linear_take_status<<<1, 1, 0, s>>>();
  if (cudaGetLastError() != cudaSuccess ||
      cudaMemcpyFromSymbolAsync(&w, ma::g_linear_taken, sizeof(w), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return MA_ERR_CUDA;
  out->code = w & 255; out->site = (w >> 8) & 255; out->cta = static_cast<uint32_t>(w >> 32); out->aux = (w >> 16) & 255;
  if (out->code == 0) return MA_OK;
  return MA_ERR_DEVICE_TIMEOUT;
}
