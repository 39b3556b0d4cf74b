// Products of e4m3 codes with a scale for each block of 128 numbers of k (gemm_q8.cu has the formula) for a moderate number of rows: one SM to a tile of 128
// rows of x by 128 or 256 rows of w, a tile's k cut into parts for a cluster of up to eight SMs.
//
// Few rows are bound by the bytes of w, and a weight has few tiles (4,096 rows are 32 of 128): cut along k, all SMs load at once.  The parts of a tile meet in
// one cluster: every SM sends each row's sums into the shared memory of the SM that adds that row up over all parts, in their order, so results do not
// depend on who was first, nothing goes through device memory, and nobody waits for a reader.
//
// As in gemm_q8_tc.cu the tensor cores hand over every block's sums and the warps add them into registers; four accumulators of 128 columns, or two of 256, take
// turns.  A tile of 128 x 128 is bound by shared memory: 32 KB a block of k arrive and are read again, 512 clocks of it beside the 256 of the products (some 600
// measured).  A tile of 256 columns reads x once for twice the products, 768 and 512 clocks, and is taken where k is long: 333 rows of 5,120 x 25,600 take 75 us in tiles
// of 128 and 61 in two parts of tiles of 256, alone in a graph (72 among calls one by one, at the power limit's clocks); its sums go where the ring was, behind one more barrier of the cluster.
//   warps 0-7        : lanes 32 (i % 4) .. + 31, columns 64 (i / 4) .. + 63 of every 128: tcgen05.ld, acc += (sx sw) * sum
//   warp 8           : producer, a TMA load of 128 rows of x and one of w a stage; what of w fits the ring is brought to L2 while the kernel in front ends
//   warp 9           : issues the products (128 x 128 or 256 x 32)
// Edges: TMA fills rows beyond M and N with zeros; stores are guarded.  Every wait is bounded; who gives up raises the error word and still comes to the
// cluster's barriers.
#include "q8.cuh"
#include "tcgen05_utils.cuh"
using namespace arle;

namespace {

constexpr int BK = 128, BM = 128;
constexpr uint32_t kTile = 128 * BK;
constexpr int kStages = 4;
constexpr int kEpilogueWarps = 8, kProducer = 8, kIssuer = 9;
constexpr uint32_t kTmemCols = 512;
constexpr int kMostParts = 8;

__device__ __forceinline__ void store_cluster(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Blocks of threads: with two blocks of columns a thread keeps 128 sums, and registers move from the third group of four warps to the first two
// (2 x 216 + 72 = 3 x 168, what the block is launched with).
template <int NB> constexpr int kThreadsOf = NB == 2 ? 384 : 320;

// NB: blocks of 128 rows of w.
template <int NB, typename OutT>
__global__ void __launch_bounds__(kThreadsOf<NB>, 1) gemm_q8_split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                    const uint8_t* sx, const float* sw, OutT* out, long ldo, int M, int N, int kb, int parts,
                                                                    int* err) {
  constexpr int BN = 128 * NB, kAccs = 4 / NB, kThreads = NB == 2 ? 384 : 320;
  constexpr uint32_t STAGE = (NB + 1) * kTile;            // w's tile, then x's
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], acc_full[kAccs], acc_empty[kAccs];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int part = (int)blockIdx.x % parts, tn = (int)blockIdx.x / parts, m0 = (int)blockIdx.y * BM, n0 = tn * BN;      // a cluster is a tile
  const int b0 = (int)((long)part * kb / parts), b1 = (int)((long)(part + 1) * kb / parts);
  const int rows = min(BM, M - m0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(smem_addr(&full_bar[s]), 1), mbar_init(smem_addr(&empty_bar[s]), 1);
    for (int a = 0; a < kAccs; ++a) mbar_init(smem_addr(&acc_full[a]), 1), mbar_init(smem_addr(&acc_empty[a]), kEpilogueWarps);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  __syncthreads();
  if (NB == 1 && parts > 1) cluster_started();             // (with two blocks of columns a barrier of its own stands in front of the stores)
  const uint32_t ring = __shfl_sync(0xffffffffu, smem_addr(tiles), 0), full0 = smem_addr(&full_bar[0]), empty0 = smem_addr(&empty_bar[0]),
                 acc_full0 = smem_addr(&acc_full[0]), acc_empty0 = smem_addr(&acc_empty[0]);
  if (warp == kProducer && elect_one())                    // to L2 and no further: a program may write w in the kernel in front
    for (int b = b0; b < min(b0 + kStages, b1); ++b) tma_prefetch_2d(&map_w, b * BK, n0);
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
  if (NB == 2 && warp >= kEpilogueWarps) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
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
        tma_load_2d(ring + s * STAGE + NB * kTile, &map_x, b * BK, m0, full0 + 8 * s);
      }
      __syncwarp();
      if (++s == kStages) s = 0, phase ^= 1;
    }
  } else if (warp == kIssuer) {
    constexpr uint32_t idesc = idesc_e4m3(BM, BN);
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
        const uint32_t blo = lo0 + s * (STAGE >> 4), alo = blo + NB * (kTile >> 4);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k) umma_e4m3(d0 + buf * BN, alo + 2 * k, blo + 2 * k, idesc, k != 0 ? 1u : 0u);
        umma_commit(acc_full0 + 8 * buf);
        umma_commit(empty0 + 8 * s);
      }
      __syncwarp();
      if (++s == kStages) s = 0, phase ^= 1;
    }
  } else if (warp < kEpilogueWarps) {
    if (NB == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
    const int half = warp >> 2, lrow = (warp & 3) * 32 + lane, blocks_n = (N + 127) / 128;
    const uint32_t lanes = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * 64);
    const uint8_t* sxr = sx + (size_t)min(m0 + lrow, M - 1) * kb;
    const float* swr[NB];
    float acc[NB][64];                                     // columns 64 half .. + 63 of every block
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      swr[h] = sw + (size_t)min(tn * NB + h, blocks_n - 1) * kb;
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[h][i] = 0.f;
    }
    const bool used = (warp & 3) * 32 < rows;              // some of this warp's rows are there
    uint32_t sx_next = sxr[b0], done = 0;
    float w_next[NB];
#pragma unroll
    for (int h = 0; h < NB; ++h) w_next[h] = swr[h][b0];
#pragma unroll 1
    for (int b = b0; b < b1; ++b, ++done) {
      const uint32_t buf = done % kAccs;
      float f[NB];
#pragma unroll
      for (int h = 0; h < NB; ++h) f[h] = __uint_as_float(sx_next << 23) * w_next[h];
      if (b + 1 < b1) {
        sx_next = sxr[b + 1];
#pragma unroll
        for (int h = 0; h < NB; ++h) w_next[h] = swr[h][b + 1];
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(acc_full0 + 8 * buf, (done / kAccs) & 1, aborted))) {
        abort_flag = 1;
        break;
      }
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        uint32_t r[2][32];
        if (used) {
          tc_fence_after();
          tmem_ld32(lanes + buf * BN + h * 128, r[0]);
          tmem_ld32(lanes + buf * BN + h * 128 + 32, r[1]);
          tmem_ld_wait(r[0]);
          tmem_ld_wait(r[1]);
          tc_fence_before();
          __syncwarp();
        }
        if (h == NB - 1 && lane == 0) asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];\n" ::"r"(acc_empty0 + 8 * buf) : "memory");
        if (used) {
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[h][i] = fmaf(__uint_as_float(r[i >> 5][i & 31]), f[h], acc[h][i]);
        }
      }
    }
    if (parts == 1) {
      if (lrow < rows && !*aborted) {
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          const int at = n0 + h * 128 + half * 64, left = N - at;
          OutT* dst = out + (size_t)(m0 + lrow) * ldo + at;
          constexpr int V = 16 / sizeof(OutT);
          if (left >= 64 && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
            for (int i = 0; i < 64 / V; ++i) {
              float v[V];
#pragma unroll
              for (int j = 0; j < V; ++j) v[j] = acc[h][i * V + j];
              store_vec<OutT, V>(dst + i * V, v);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i < left) dst[i] = from_f32<OutT>(acc[h][i]);
          }
        }
      }
    } else {
      // Row l is added up by SM l % parts of the cluster, as its row j = l / parts: 512 NB bytes from each part as pieces of 16 bytes, piece p at p ^ (j % 8), so
      // that eight rows' pieces lie in different banks.  Behind the ring, or in it when no SM of the cluster has use for it any more.
      if (NB == 2) cluster_sync_all();
      else cluster_all_started();
      const uint32_t slots = (uint32_t)((rows + parts - 1) / parts);
      if (lrow < rows) {
        const uint32_t j = (uint32_t)(lrow / parts),
                       to = map_to_rank(ring + (NB == 2 ? 0u : kStages * STAGE) + ((uint32_t)part * slots + j) * (512 * NB), (uint32_t)(lrow % parts));
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int p = 0; p < 16; ++p)
            store_cluster(to + 16 * (uint32_t)((h * 32 + half * 16 + p) ^ (j & 7)), make_float4(acc[h][4 * p], acc[h][4 * p + 1], acc[h][4 * p + 2], acc[h][4 * p + 3]));
      }
    }
  }
  if (parts > 1) {
    if (warp >= kEpilogueWarps) {
      if (NB == 2) cluster_sync_all();
      else cluster_all_started();
    }
    cluster_sync_all();
    const int slots = (rows + parts - 1) / parts;
    const unsigned char* mine = tiles + (NB == 2 ? 0u : kStages * STAGE);
    if (!*aborted)
      for (int j = warp; j * parts + part < rows; j += kThreads / 32) {
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          const int col = n0 + h * 128 + 4 * lane;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int p = 0; p < parts; ++p) {
            const float4 o = *reinterpret_cast<const float4*>(mine + ((size_t)p * slots + j) * (512 * NB) + 16 * ((h * 32 + lane) ^ (j & 7)));
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
          }
          OutT* dst = out + (size_t)(m0 + j * parts + part) * ldo + col;
          const float vv[4] = {v.x, v.y, v.z, v.w};
          if (col + 4 <= N && ((uintptr_t)dst % (4 * sizeof(OutT))) == 0) {
            store_vec<OutT, 4>(dst, vv);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (col + i < N) dst[i] = from_f32<OutT>(vv[i]);
          }
        }
      }
  }
  // copies may still be under way where a wait ran out: every one is counted on a barrier of this SM
  __syncthreads();
  if (*aborted && warp == kProducer && lane == 0)
    for (int s = 0; s < kStages; ++s) mbar_wait_plain(smem_addr(&full_bar[s]), 0), mbar_wait_plain(smem_addr(&full_bar[s]), 1);
  tc_fence_before();
  __syncthreads();
  pdl_launch_dependents();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && abort_flag && err) atomicExch(err, 4);
}

template <int NB> constexpr size_t kSharedBytes = (size_t)kStages * (NB + 1) * kTile + (NB == 2 ? 0 : (size_t)(BM + kMostParts) * 512) + 1024;
static_assert((size_t)(BM + kMostParts) * 1024 <= (size_t)kStages * 3 * kTile, "the sums of 256 columns fit the ring");

template <int NB, typename OutT>
int launch_split(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, int parts, int* err, cudaStream_t s) {
  CUtensorMap mx, mw;
  int rc = tensor_map_2d_u8(x, M, kb * BK, BM, &mx);
  if (rc) return rc;
  rc = tensor_map_2d_u8(w, N, kb * BK, 128 * NB, &mw);
  if (rc) return rc;
  const long tiles_n = ((long)N + 128 * NB - 1) / (128 * NB), tiles_m = ((long)M + BM - 1) / BM;
  if (tiles_m > 65535 || tiles_n * parts > 0x7fffffffl) return ARLE_E_UNSUPPORTED;
  auto kern = gemm_q8_split_kernel<NB, OutT>;
  static SharedLimit limit;
  const cudaError_t raised = limit.raise((const void*)kern, kSharedBytes<NB>);
  if (raised != cudaSuccess) return (int)raised;
  const cudaError_t e = launch_early(kern, dim3((unsigned)(tiles_n * parts), (unsigned)tiles_m), dim3(kThreadsOf<NB>), kSharedBytes<NB>, s, parts, mx, mw,
                                     (const uint8_t*)sx, sw, (OutT*)out, ldo, M, N, kb, parts, err);
  if (e != cudaSuccess) return (int)e;
  return launch_status();
}

template <typename OutT>
int product(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, int parts, int nb, int* err, cudaStream_t s) {
  return nb == 2 ? launch_split<2, OutT>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s) : launch_split<1, OutT>(x, sx, w, sw, out, ldo, M, N, kb, parts, err, s);
}

}  // namespace

// As arle_gemm_q8_pair; parts: 1 to 8 (at most kb), the SMs that share a tile's k; nb: 1 or 2, blocks of 128 rows of w to a tile.  err: set to 4 if a wait ran out.
ARLE_API int arle_gemm_q8_split(const void* x, const void* sx, const void* w, const float* sw, void* out, int out_dtype, long ldo, int M, int N, int kb, int parts,
                                int nb, int* err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (kb <= 0 || kb > (1 << 23) || parts < 1 || parts > kMostParts || parts > kb || nb < 1 || nb > 2 || (((uintptr_t)x | (uintptr_t)w) & 15)) return ARLE_E_BADARG;
  if (out_dtype == 0) return product<float>(x, sx, w, sw, out, ldo, M, N, kb, parts, nb, err, s);
  if (out_dtype == 1) return product<__nv_bfloat16>(x, sx, w, sw, out, ldo, M, N, kb, parts, nb, err, s);
  return ARLE_E_BADARG;
}

// How many clusters of `parts` SMs a device runs at a time (an SM holds one block); negative: an error.  The current device stays what it is.
ARLE_API int arle_gemm_q8_split_clusters(int parts, int device) {
  if (parts < 1 || parts > kMostParts) return ARLE_E_BADARG;
  int was = 0;
  if (cudaGetDevice(&was) != cudaSuccess || (device != was && cudaSetDevice(device) != cudaSuccess)) return -1;
  auto kern = gemm_q8_split_kernel<1, float>;
  int n = -1;
  if (cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedBytes<1>) == cudaSuccess) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreadsOf<1>), cfg.gridDim = dim3(parts), cfg.dynamicSmemBytes = kSharedBytes<1>, cfg.attrs = &attr, cfg.numAttrs = 1;
    int found = 0;
    if (cudaOccupancyMaxActiveClusters(&found, kern, &cfg) == cudaSuccess) n = found;
  }
  if (device != was && cudaSetDevice(was) != cudaSuccess) return -1;
  return n;
}
