// Products of e4m3 codes with a scale for each block of 128 numbers of k (gemm_q8.cu has the formula) for a batch of decoded tokens (9 to 64 rows), bound by the
// bytes of w: a block owns 128 rows of w, which are the lanes of the tensor cores' accumulators, and all rows of x, which are their columns; a tile's k is cut into
// parts for a cluster of up to eight blocks.
//
// Two blocks share an SM (100 KB and 192 threads each), so one loads while the other starts, hands over or ends, and their first tiles of w are brought to L2 while the
// kernel in front ends (and loaded behind the wait for it, since it may have written them: no slower from 16 rows on than loaded in front of it).  The next kernel may start when a block has joined its parts: norms, codes and the four
// products of a layer of 8B sizes take 55.4 us for 16 rows and 67.6 for 64 when it may start at once, 53.2 and 63.9 so.  The parts of a tile meet in one cluster: each sends a row of x's
// sums into the shared memory of the block that adds that row up over all parts, in their order, so results do not depend on who was first.
//   warps 0-3 : lanes 32 i .. + 31: tcgen05.ld, acc[column] += (sx[column] sw) * sum; those factors lie in shared memory, 256 at a time
//   warp 4    : producer, TMA loads of 128 rows of w and ROWS rows of x a stage
//   warp 5    : issues the products (128 x ROWS x 32); four accumulators take turns
// Edges: TMA fills rows beyond M and N with zeros; stores are guarded.  Every wait is bounded; who gives up raises the error word and still comes to the
// cluster's barrier.
#include "q8.cuh"
#include "tcgen05_utils.cuh"
using namespace arle;

namespace {

constexpr int BK = 128, BN = 128;                          // codes of a stage; rows of w
constexpr uint32_t kTile = BN * BK;
constexpr int kAccs = 4, kAddWarps = 4, kProducer = 4, kIssuer = 5, kThreads = 192;
constexpr int kMostParts = 8;
template <int ROWS> constexpr int kScaled = 256 / ROWS;      // blocks of k whose factors are at hand
template <int ROWS> constexpr int kStagesOf = ROWS == 64 ? 3 : 4;
// The sums that a block adds up: groups of four rows from every part, at most this many in all.  (64 rows are 16 groups: 18 from three or six parts, 20 and 21
// from five and seven, for which there is no room beside two blocks' rings.)
template <int ROWS> constexpr int kMostGroups = ROWS == 64 ? 18 : ROWS == 32 ? 14 : 8;
template <int ROWS> constexpr size_t kSharedBytes =
    (size_t)kStagesOf<ROWS> * (kTile + ROWS * BK) + (size_t)kMostGroups<ROWS> * 2048 + 2 * kScaled<ROWS> * ROWS * sizeof(float) + 1024;

__device__ __forceinline__ void store_cluster(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void bar_adders() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }

template <int C> __device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[C]);
template <> __device__ __forceinline__ void tmem_ld<32>(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld32(taddr, r);
  tmem_ld_wait(r);
}
template <> __device__ __forceinline__ void tmem_ld<16>(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr) : "memory");
}

template <int ROWS, typename OutT>
__global__ void __launch_bounds__(kThreads, 2) gemm_q8_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                  const uint8_t* sx, const float* sw, OutT* out, long ldo, int M, int N, int kb, int parts,
                                                                  int* err) {
  constexpr int STAGES = kStagesOf<ROWS>, SCALED = 256 / ROWS, CHUNK = ROWS < 32 ? ROWS : 32;
  constexpr uint32_t STAGE = kTile + ROWS * BK, kTmemCols = kAccs * ROWS;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  float4* sums = reinterpret_cast<float4*>(tiles + STAGES * STAGE);                      // [part][group of four rows][128]
  float* factors = reinterpret_cast<float*>(tiles + STAGES * STAGE + (size_t)kMostGroups<ROWS> * 2048);        // [2][block of k][row]: sx sw
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[kAccs], acc_empty[kAccs];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int part = (int)blockIdx.x % parts, tn = (int)blockIdx.x / parts, n0 = tn * BN;                  // a cluster is a tile
  const int b0 = (int)((long)part * kb / parts), b1 = (int)((long)(part + 1) * kb / parts);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_addr(&full_bar[s]), 1), mbar_init(smem_addr(&empty_bar[s]), 1);
    for (int a = 0; a < kAccs; ++a) mbar_init(smem_addr(&acc_full[a]), 1), mbar_init(smem_addr(&acc_empty[a]), kAddWarps);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  __syncthreads();
  if (parts > 1) cluster_started();
  const uint32_t ring = __shfl_sync(0xffffffffu, smem_addr(tiles), 0), full0 = smem_addr(&full_bar[0]), empty0 = smem_addr(&empty_bar[0]),
                 acc_full0 = smem_addr(&acc_full[0]), acc_empty0 = smem_addr(&acc_empty[0]);
  if (warp == kProducer && elect_one())                    // to L2 and no further: a program may write w in the kernel in front
    for (int b = b0; b < min(b0 + STAGES, b1); ++b) tma_prefetch_2d(&map_w, b * BK, n0);
  __syncwarp();
  // Tensor memory is asked for when the kernel in front has ended, and the next kernel may start when it is had (in fact far later): a block that held some while it
  // waited for one that still has to get it on the same SM would wait for good.
  pdl_wait();
  if (warp == kIssuer) {
    tmem_alloc(smem_addr(&tmem_base_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  const volatile int* aborted = &abort_flag;
  float acc[ROWS];

  if (warp == kProducer) {
    int s = 0;
    uint32_t phase = 1;
    for (int b = b0; b < b1; ++b) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(empty0 + 8 * s, phase, aborted))) {
        abort_flag = 1;
        break;
      }
      if (elect_one()) {
        mbar_expect_tx(full0 + 8 * s, STAGE);
        tma_load_2d(ring + s * STAGE, &map_w, b * BK, n0, full0 + 8 * s);
        tma_load_2d(ring + s * STAGE + kTile, &map_x, b * BK, 0, full0 + 8 * s);
      }
      __syncwarp();
      if (++s == STAGES) s = 0, phase ^= 1;
    }
  } else if (warp == kIssuer) {
    constexpr uint32_t idesc = idesc_e4m3(BN, ROWS);
    const uint32_t d0 = __shfl_sync(0xffffffffu, tmem_base, 0), lo0 = smem_desc_sw128_lo(ring);
    int s = 0;
    uint32_t phase = 0, done = 0;
    for (int b = b0; b < b1; ++b, ++done) {
      const uint32_t buf = done % kAccs;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(full0 + 8 * s, phase, aborted) &&
                                       mbar_wait_bounded(acc_empty0 + 8 * buf, ((done / kAccs) & 1) ^ 1, aborted))) {
        abort_flag = 1;
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint32_t alo = lo0 + s * (STAGE >> 4), blo = alo + (kTile >> 4);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k) umma_e4m3(d0 + buf * ROWS, alo + 2 * k, blo + 2 * k, idesc, k != 0 ? 1u : 0u);
        umma_commit(acc_full0 + 8 * buf);
        umma_commit(empty0 + 8 * s);
      }
      __syncwarp();
      if (++s == STAGES) s = 0, phase ^= 1;
    }
  } else {
    const uint32_t lanes = tmem_base + ((uint32_t)(warp * 32) << 16);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) acc[i] = 0.f;
    // The factors of SCALED blocks lie in shared memory, those of the next ones are on their way in registers.  A thread has one block's for two rows.
    const int at = threadIdx.x % SCALED, m_first = threadIdx.x / SCALED;
    constexpr int MINE = 2, STEP = 128 / SCALED;
    uint8_t e_next[MINE];
    float w_next = 0.f;
    auto ask = [&](int b) {
      const int mine = min(b + at, b1 - 1);
      w_next = sw[(size_t)tn * kb + mine];
#pragma unroll
      for (int i = 0; i < MINE; ++i) e_next[i] = sx[(size_t)min(m_first + STEP * i, M - 1) * kb + mine];
    };
    ask(b0);
    uint32_t done = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b, ++done) {
      const uint32_t buf = done % kAccs;
      float* fs = factors + (done / SCALED % 2) * (SCALED * ROWS);
      if (done % SCALED == 0) {                           // (who still reads the other half has not come to this barrier)
#pragma unroll
        for (int i = 0; i < MINE; ++i) fs[at * ROWS + m_first + STEP * i] = __uint_as_float((uint32_t)e_next[i] << 23) * w_next;
        bar_adders();
        if (b + SCALED < b1) ask(b + SCALED);
      }
      const float4* f4 = reinterpret_cast<const float4*>(fs + (done % SCALED) * ROWS);
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(acc_full0 + 8 * buf, (done / kAccs) & 1, aborted))) {
        abort_flag = 1;
        // another warp's poll may have succeeded: this one still comes to the barriers that are left, which have no limit
        for (uint32_t later = done + 1; later < (uint32_t)(b1 - b0); ++later)
          if (later % SCALED == 0) bar_adders();
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < ROWS / CHUNK; ++c) {
        uint32_t r[CHUNK];
        tmem_ld<CHUNK>(lanes + buf * ROWS + c * CHUNK, r);
        if (c == ROWS / CHUNK - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];\n" ::"r"(acc_empty0 + 8 * buf) : "memory");
        }
#pragma unroll
        for (int i = 0; i < CHUNK; i += 4) {
          const float4 f = f4[(c * CHUNK + i) / 4];
          float* a = acc + c * CHUNK + i;
          a[0] = fmaf(__uint_as_float(r[i]), f.x, a[0]), a[1] = fmaf(__uint_as_float(r[i + 1]), f.y, a[1]);
          a[2] = fmaf(__uint_as_float(r[i + 2]), f.z, a[2]), a[3] = fmaf(__uint_as_float(r[i + 3]), f.w, a[3]);
        }
      }
    }
  }
  // copies may still be under way where a wait ran out: every one is counted on a barrier of this block
  __syncthreads();
  if (*aborted && warp == kProducer && lane == 0)
    for (int s = 0; s < STAGES; ++s) mbar_wait_plain(smem_addr(&full_bar[s]), 0), mbar_wait_plain(smem_addr(&full_bar[s]), 1);
  if (*aborted) __syncthreads();

  // the group of rows 4q .. 4q + 3 is added up by block q % parts of the cluster, as its group q / parts
  const int slots = (ROWS / 4 + parts - 1) / parts;
  if (parts > 1) {
    cluster_all_started();
    if (warp < kAddWarps) {
      uint32_t to = 0, slot = smem_addr(sums) + ((uint32_t)(part * slots) * 128 + threadIdx.x) * 16;
#pragma unroll
      for (int q = 0; q < ROWS / 4; ++q) {
        if (4 * q < M) store_cluster(map_to_rank(slot, to), acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        if (++to == (uint32_t)parts) to = 0, slot += 2048;
      }
    }
    cluster_sync_all();
  }
  if (warp < kAddWarps && !*aborted && n0 + (int)threadIdx.x < N) {
    OutT* dst = out + n0 + threadIdx.x;
    if (parts == 1) {
#pragma unroll
      for (int m = 0; m < ROWS; ++m)
        if (m < M) dst[(size_t)m * ldo] = from_f32<OutT>(acc[m]);
    } else {
      for (int j = 0, m = 4 * part; m < M; ++j, m += 4 * parts) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int p = 0; p < kMostParts; ++p)
          if (p < parts) {
            const float4 o = sums[(p * slots + j) * 128 + threadIdx.x];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
          }
        OutT* d = dst + (size_t)m * ldo;
        d[0] = from_f32<OutT>(v.x);
        if (m + 1 < M) d[ldo] = from_f32<OutT>(v.y);
        if (m + 2 < M) d[2 * ldo] = from_f32<OutT>(v.z);
        if (m + 3 < M) d[3 * ldo] = from_f32<OutT>(v.w);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  pdl_launch_dependents();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && abort_flag && err) atomicExch(err, 5);
}

template <int ROWS, typename OutT>
int launch_few(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, int parts, int* err, cudaStream_t s) {
  CUtensorMap mx, mw;
  int rc = tensor_map_2d_u8(x, M, kb * BK, ROWS, &mx);
  if (rc) return rc;
  rc = tensor_map_2d_u8(w, N, kb * BK, BN, &mw);
  if (rc) return rc;
  const long blocks = ((long)N + BN - 1) / BN * parts;
  if (blocks > 0x7fffffffl) return ARLE_E_UNSUPPORTED;
  auto kern = gemm_q8_few_kernel<ROWS, OutT>;
  static SharedLimit limit;
  const cudaError_t raised = limit.raise((const void*)kern, kSharedBytes<ROWS>, true);
  if (raised != cudaSuccess) return (int)raised;
  const cudaError_t e = launch_early(kern, dim3((unsigned)blocks), dim3(kThreads), kSharedBytes<ROWS>, s, parts, mx, mw, (const uint8_t*)sx, sw, (OutT*)out, ldo, M, N,
                                     kb, parts, err);
  if (e != cudaSuccess) return (int)e;
  return launch_status();
}

template <typename OutT>
int product(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, int parts, int* err, cudaStream_t s) {
  if (M <= 16) return launch_few<16, OutT>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
  if (M <= 32) return launch_few<32, OutT>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
  return launch_few<64, OutT>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
}

}  // namespace

// As arle_gemm_q8_pair, for M up to 64; parts: 1 to 8 (at most kb), the blocks that share a tile's k.  err: set to 5 if a wait ran out.
ARLE_API int arle_gemm_q8_few(const void* x, const void* sx, const void* w, const float* sw, void* out, int out_dtype, long ldo, int M, int N, int kb, int parts,
                              int* err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (M > 64 || (M > 32 && (parts == 5 || parts == 7))) return ARLE_E_UNSUPPORTED;
  if (kb <= 0 || kb > (1 << 23) || parts < 1 || parts > kMostParts || parts > kb || (((uintptr_t)x | (uintptr_t)w) & 15)) return ARLE_E_BADARG;
  if (out_dtype == 0) return product<float>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
  if (out_dtype == 1) return product<__nv_bfloat16>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
  return ARLE_E_BADARG;
}
