// Products of e4m3 codes with a scale for each block of 128 numbers of k (gemm_q8.cu has the formula), on the tensor cores of sm_100a, for many rows:
// two SMs to a tile of 256 rows of x by 256 rows of w.
//
// A scale that changes every 128 numbers of k cannot be applied behind the whole sum, so the tensor cores hand over every block's sum: an accumulator of 128
// lanes x 256 columns is one block of k (four tcgen05.mma of 32), two of them take turns in the 512 columns of tensor memory, and the epilogue warps add
// block after block into registers, acc += (sx[row] sw[block of columns]) * sum.  A lane is a row of x and 128 columns are one block of w, so that
// factor is one number a thread and 128 columns.  A block's products take the tensor cores 512 clocks, reading and adding its sums takes the warps some 270,
// and a block takes 670 to 790 (4,096 rows of 4,096 x 12,288).  With two accumulators in turn the 270 should be hidden; what the rest waits for has not been measured.
// 4,096 rows of 4,096 x 12,288 179 us alone (2.3 PFLOP/s), 209 to 212 back to back, where 1,000 W hold the clock at 1.4 GHz; gated, 24,576 x 4,096, 350 and 408.
//
// Per CTA, by warp:
//   warps 0-7        : epilogue of the CTA's 128 rows; warp i reads lanes 32 (i % 4) .. + 31, of columns 64 h .. 64 h + 63 and 128 + 64 h .. (h = i / 4).  Gated,
//                      columns 0-127 are gates and 128-255 what they multiply, so a thread holds both numbers of its 64 results, and the two threads of
//                      a row exchange nothing but their largest number: the 128 results of a tile are one group of codes.
//   warp 8, one lane : producer, a TMA load of 128 rows of x and one of 128 rows of w (16 KB each, 128-byte swizzle) a stage, counted on the first CTA's barrier
//   warp 9, one lane : in the first CTA, issues the products of the pair (256 x 256 x 32) and hands stages and accumulators on by commits
// Edges: TMA fills rows beyond M and N with zeros; stores are guarded.  Every wait is bounded (see gemm_tcgen05_pair.cu, whose way of giving up this is).
#include "q8.cuh"
#include "tcgen05_utils.cuh"
using namespace arle;

namespace {

constexpr int BK = 128;                          // codes = bytes: one swizzle span, one block of scales
constexpr int BM = 128, BN = 256;                // rows of x per CTA, rows of w per pair
constexpr uint32_t kTile = 128 * BK;             // bytes of either operand's part of a stage
constexpr int kEpilogueWarps = 8, kProducer = 8, kIssuer = 9, kThreads = 384;      // (warps 10 and 11 fill up the third group of four)
constexpr uint32_t kTmemCols = 512;

// acc (two float32 numbers) += {d0, d1} * f
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t d0, uint32_t d1, uint64_t f) {
  asm volatile("{\n.reg .b64 d;\nmov.b64 d, {%1, %2};\nfma.rn.f32x2 %0, d, %3, %0;\n}\n" : "+l"(acc) : "r"(d0), "r"(d1), "l"(f));
}
__device__ __forceinline__ uint64_t both(float f) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};\n" : "=l"(r) : "f"(f));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
// Registers move from the third group of four warps to the first two, which keep 128 sums a thread: 2 x 216 + 72 = 3 x 168, what the block is launched with.
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n"); }
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n"); }

// An arrival that orders no memory accesses: what it hands over is tensor memory, whose reads are done when tcgen05.wait::ld returns.  (A release by all sixteen
// warps for every block of k waits for their loads of scales: 454 us instead of 228 for 4,096 rows of 4,096 x 12,288.)
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void bar_pair(int id) { asm volatile("bar.sync %0, 64;\n" ::"r"(id) : "memory"); }

// 2 C numbers of a row to out[0 .. 2 C), of which `left` are there.
template <int C, typename OutT>
__device__ __forceinline__ void store_row(OutT* dst, const uint64_t (&acc)[C], int left) {
  constexpr int V = 16 / sizeof(OutT);
  if (left >= 2 * C && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 2 * C / V; ++i) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 p = halves(acc[i * (V / 2) + j]);
        v[2 * j] = p.x, v[2 * j + 1] = p.y;
      }
      store_vec<OutT, V>(dst + i * V, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const float2 p = halves(acc[i]);
      if (2 * i < left) dst[2 * i] = from_f32<OutT>(p.x);
      if (2 * i + 1 < left) dst[2 * i + 1] = from_f32<OutT>(p.y);
    }
  }
}

template <int STAGES, bool GATED, typename OutT>
__global__ void __launch_bounds__(kThreads, 1) gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                   const uint8_t* sx, const float* sw, OutT* out, long ldo, uint8_t* out_scales, int M,
                                                                   int N, int kb, int act, int* err) {
  pdl_wait();
  constexpr uint32_t STAGE = 2 * kTile;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[STAGES];      // first CTA's: both CTAs' copies of the stage have landed
  __shared__ __align__(8) uint64_t empty_bar[STAGES];     // each CTA's: the products have read the stage
  __shared__ __align__(8) uint64_t acc_full[2];           // each CTA's: a block's sums are there
  __shared__ __align__(8) uint64_t acc_empty[2];          // first CTA's: both CTAs' epilogues have read them
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ uint32_t most_s[2][BM];

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = (int)(blockIdx.x >> 1), npairs = (int)(gridDim.x >> 1);
  const int tiles_m = (M + 2 * BM - 1) / (2 * BM), tiles_n = (N + BN - 1) / BN;
  const int num_tiles = tiles_m * tiles_n;
  // bands of kBand rows of tiles, inside a band the row index fastest: pairs that run together share a few tiles of w and kBand of x in L2
  constexpr int kBand = 8;
  auto tile_at = [&](int t, int& tm, int& tn) {
    const int band = t / (kBand * tiles_n);
    const int rows_here = min(kBand, tiles_m - band * kBand);
    const int in_band = t - band * kBand * tiles_n;
    tm = band * kBand + in_band % rows_here;
    tn = in_band / rows_here;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_addr(&full_bar[s]), 1);
      mbar_init(smem_addr(&empty_bar[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&acc_full[b]), 1);
      mbar_init(smem_addr(&acc_empty[b]), 2 * kEpilogueWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == kIssuer) {
    tmem_alloc_pair(smem_addr(&tmem_base_slot), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // the partner's barriers exist before anything arrives on them
  pdl_launch_dependents();                                 // with its tensor memory in hand: who starts beside it may want some too
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  const volatile int* aborted = &abort_flag;

  if (warp >= kEpilogueWarps) {
    fewer_registers();
    const uint32_t ring = __shfl_sync(0xffffffffu, smem_addr(tiles), 0), full0 = smem_addr(&full_bar[0]), empty0 = smem_addr(&empty_bar[0]);
    if (warp == kProducer) {
      const uint32_t full_leader = map_to_rank(full0, 0);
      int s = 0;
      uint32_t phase = 1;
      for (int t = pair; t < num_tiles && !*aborted; t += npairs) {
        int tm, tn;
        tile_at(t, tm, tn);
        const int m0 = tm * 2 * BM + (int)rank * BM, n0 = tn * BN + (int)rank * 128;
        for (int b = 0; b < kb; ++b) {
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(empty0 + 8 * s, phase, aborted))) {
            abort_flag = 1;
            break;
          }
          if (elect_one()) {
            const uint32_t bar = full_leader + 8 * s, dst = ring + s * STAGE;
            if (leader) mbar_expect_tx(full0 + 8 * s, 2 * STAGE);           // the bytes of both CTAs
            tma_load_2d_pair(dst, &map_x, b * BK, m0, bar);
            tma_load_2d_pair(dst + kTile, &map_w, b * BK, n0, bar);
          }
          __syncwarp();
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
    } else if (warp == kIssuer && leader) {
      constexpr uint32_t idesc = idesc_e4m3(2 * BM, BN);
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem_base, 0), lo0 = smem_desc_sw128_lo(ring), acc_full0 = smem_addr(&acc_full[0]),
                     acc_empty0 = smem_addr(&acc_empty[0]);
      int s = 0;
      uint32_t phase = 0, done = 0;                        // done: blocks of k over all tiles; accumulator done % 2
      for (int t = pair; t < num_tiles && !*aborted; t += npairs) {
        for (int b = 0; b < kb; ++b, ++done) {
          const uint32_t buf = done & 1;
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(full0 + 8 * s, phase, aborted) &&
                                           mbar_wait_bounded(acc_empty0 + 8 * buf, ((done >> 1) & 1) ^ 1, aborted))) {
            abort_flag = 1;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t alo = lo0 + s * (STAGE >> 4), blo = alo + (kTile >> 4);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k) umma_e4m3_pair(d0 + buf * BN, alo + 2 * k, blo + 2 * k, idesc, k != 0 ? 1u : 0u);
            umma_commit_both(acc_full0 + 8 * buf);
            umma_commit_both(empty0 + 8 * s);
          }
          __syncwarp();
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
    }
  } else {
    more_registers();
    const int half = warp >> 2, lrow = (warp & 3) * 32 + lane, blocks_n = (N + BK - 1) / BK;
    const uint32_t acc_full0 = smem_addr(&acc_full[0]), acc_empty_leader = map_to_rank(smem_addr(&acc_empty[0]), 0);
    const uint32_t lanes = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * 64);
    uint32_t done = 0;
    bool lost = false;
    for (int t = pair; t < num_tiles && !lost; t += npairs) {
      int tm, tn;
      tile_at(t, tm, tn);
      const int row = tm * 2 * BM + (int)rank * BM + lrow, n0 = tn * BN;
      const uint8_t* sxr = sx + (size_t)min(row, M - 1) * kb;
      const float* sw0 = sw + (size_t)min(2 * tn, blocks_n - 1) * kb;
      const float* sw1 = sw + (size_t)min(2 * tn + 1, blocks_n - 1) * kb;
      uint64_t acc[2][32];                                 // columns 64 half .. + 63 and 128 + 64 half .. + 63
#pragma unroll
      for (int i = 0; i < 32; ++i) acc[0][i] = acc[1][i] = 0;
      uint32_t sx_next = sxr[0];
      float w0_next = sw0[0], w1_next = sw1[0];
      auto block = [&](uint32_t src, uint32_t full, uint32_t phase, uint32_t empty, uint64_t f0, uint64_t f1) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(full, phase, aborted))) return false;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[2][32];
          tmem_ld32(src + h * 128, r[0]);
          tmem_ld32(src + h * 128 + 32, r[1]);
          tmem_ld_wait(r[0]);
          asm volatile("" : "+r"(r[1][0]), "+r"(r[1][1]), "+r"(r[1][2]), "+r"(r[1][3]), "+r"(r[1][4]), "+r"(r[1][5]), "+r"(r[1][6]), "+r"(r[1][7]), "+r"(r[1][8]), "+r"(r[1][9]), "+r"(r[1][10]), "+r"(r[1][11]), "+r"(r[1][12]), "+r"(r[1][13]), "+r"(r[1][14]), "+r"(r[1][15]), "+r"(r[1][16]), "+r"(r[1][17]), "+r"(r[1][18]), "+r"(r[1][19]), "+r"(r[1][20]), "+r"(r[1][21]), "+r"(r[1][22]), "+r"(r[1][23]), "+r"(r[1][24]), "+r"(r[1][25]), "+r"(r[1][26]), "+r"(r[1][27]), "+r"(r[1][28]), "+r"(r[1][29]), "+r"(r[1][30]), "+r"(r[1][31]) :: "memory");
          if (h == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_relaxed(empty);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) fma2(acc[h][i], r[i >> 4][2 * (i & 15)], r[i >> 4][2 * (i & 15) + 1], h ? f1 : f0);
        }
        return true;
      };
#pragma unroll 1
      for (int b = 0; b < kb; ++b, ++done) {
        const uint32_t buf = done & 1;
        const float fx = __uint_as_float(sx_next << 23);
        const uint64_t f0 = both(fx * w0_next), f1 = both(fx * w1_next);
        if (b + 1 < kb) sx_next = sxr[b + 1], w0_next = sw0[b + 1], w1_next = sw1[b + 1];
        if (!block(lanes + buf * BN, acc_full0 + 8 * buf, (done >> 1) & 1, acc_empty_leader + 8 * buf, f0, f1)) {
          abort_flag = 1;
          lost = true;
          break;
        }
      }
      if (lost) {
        if constexpr (GATED)                               // the other half's warp may go on: this one still comes to the barriers that the two share
          for (; t < num_tiles; t += npairs) bar_pair(1 + (warp & 3)), bar_pair(1 + (warp & 3));
        break;
      }
      if constexpr (GATED) {
        // the row's largest result is known to both of its threads after one exchange
        uint32_t most = 0;
        auto gate = [&](auto act_of) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 g = halves(acc[0][i]), u = halves(acc[1][i]);
            const float y0 = act_of(g.x) * u.x, y1 = act_of(g.y) * u.y;
            asm("mov.b64 %0, {%1, %2};\n" : "=l"(acc[0][i]) : "f"(y0), "f"(y1));
            most = max(most, max(abs_bits(y0), abs_bits(y1)));
          }
        };
        if (act == 0) gate([](float g) { return q8_silu(g); });
        else gate([](float g) { return q8_gelu_tanh(g); });
        if (__any_sync(0xffffffffu, most >= kInfBits)) {   // numbers that are not finite become NaN and do not count
          most = 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 y = halves(acc[0][i]);
            most = max(most, max(finite_bits(y.x), finite_bits(y.y)));
            asm("mov.b64 %0, {%1, %2};\n" : "=l"(acc[0][i]) : "f"(finite_or_nan(y.x)), "f"(finite_or_nan(y.y)));
          }
        }
        most_s[half][lrow] = most;
        bar_pair(1 + (warp & 3));
        most = max(most, most_s[half ^ 1][lrow]);
        bar_pair(1 + (warp & 3));                          // read by both before the next tile writes
        const float s = q8_scale(__uint_as_float(most)), inv = inverse_scale(s);
        if (row < M) {
          uint8_t* dst = reinterpret_cast<uint8_t*>(out) + (size_t)row * ldo + (size_t)tn * 128 + half * 64;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 a = halves(acc[0][8 * i + 2 * j]), c = halves(acc[0][8 * i + 2 * j + 1]);
              w[j] = q8_codes4(a.x * inv, a.y * inv, c.x * inv, c.y * inv);
            }
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (half == 0) out_scales[(size_t)row * tiles_n + tn] = exponent_byte(s);
        }
      } else {
        if (row < M) {
          OutT* dst = out + (size_t)row * ldo + n0 + half * 64;
          store_row<32, OutT>(dst, acc[0], N - n0 - half * 64);
          store_row<32, OutT>(dst + 128, acc[1], N - n0 - 128 - half * 64);
        }
      }
    }
  }
  // where a wait ran out, copies may still be under way into the pair's shared memory: they are counted on the first CTA's barriers, and it waits (bounded)
  __syncthreads();
  if (warp == kProducer && lane == 0 && leader && *aborted)
    for (int s = 0; s < STAGES; ++s) mbar_wait_plain(smem_addr(&full_bar[s]), 0), mbar_wait_plain(smem_addr(&full_bar[s]), 1);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // neither CTA frees tensor memory the other's products may still write
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && abort_flag && err) atomicExch(err, 3);
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <bool GATED, typename OutT>
int launch_pair(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, void* out_scales, int M, int N, int kb, int act, int* err,
                cudaStream_t s) {
  constexpr int STAGES = 6;
  CUtensorMap mx, mw;
  int rc = tensor_map_2d_u8(x, M, kb * BK, BM, &mx);
  if (rc) return rc;
  rc = tensor_map_2d_u8(w, N, kb * BK, 128, &mw);
  if (rc) return rc;
  const size_t smem = (size_t)STAGES * 2 * kTile + 1024;
  auto kern = gemm_q8_pair_kernel<STAGES, GATED, OutT>;
  static SharedLimit limit;
  const cudaError_t raised = limit.raise((const void*)kern, smem);
  if (raised != cudaSuccess) return (int)raised;
  const long long num_tiles = (long long)((N + BN - 1) / BN) * ((M + 2 * BM - 1) / (2 * BM));
  if (num_tiles > 0x7fffffffll) return ARLE_E_UNSUPPORTED;
  long long pairs = sm_count() / 2;
  if (num_tiles < pairs) pairs = num_tiles;
  const cudaError_t e = launch_kernel(kern, dim3((unsigned)(2 * pairs)), dim3(kThreads), smem, s, 2, mx, mw, (const uint8_t*)sx, sw, (OutT*)out, ldo,
                                      (uint8_t*)out_scales, M, N, kb, act, err);
  if (e != cudaSuccess) return (int)e;
  return launch_status();
}

}  // namespace

// x [M, 128 kb], sx [M, kb], w [N, 128 kb], sw [ceil(N / 128), kb], out [M, N] of rows ldo apart (0 float32, 1 bfloat16).  err: set to 3 if a wait ran out.
ARLE_API int arle_gemm_q8_pair(const void* x, const void* sx, const void* w, const float* sw, void* out, int out_dtype, long ldo, int M, int N, int kb, int* err,
                               cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (kb <= 0 || kb > (1 << 23) || (((uintptr_t)x | (uintptr_t)w) & 15)) return ARLE_E_BADARG;
  if (out_dtype == 0) return launch_pair<false, float>(x, sx, w, sw, out, ldo, nullptr, M, N, kb, 0, err, s);
  if (out_dtype == 1) return launch_pair<false, __nv_bfloat16>(x, sx, w, sw, out, ldo, nullptr, M, N, kb, 0, err, s);
  return ARLE_E_BADARG;
}

// w [256 nb, 128 kb]: 128 rows of the gate, 128 of the other, and so on; codes [M, 128 nb] and scales [M, nb] of act(gate) * up; act 0 silu, 1 the tanh form of gelu.
ARLE_API int arle_gemm_q8_pair_gated(const void* x, const void* sx, const void* w, const float* sw, void* codes, void* scales, int M, int nb, int kb, int act,
                                     int* err, cudaStream_t s) {
  if (M <= 0 || nb <= 0) return 0;
  if (kb <= 0 || kb > (1 << 23) || nb > (1 << 22) || act < 0 || act > 1 || (((uintptr_t)x | (uintptr_t)w | (uintptr_t)codes) & 15)) return ARLE_E_BADARG;
  return launch_pair<true, uint8_t>(x, sx, w, sw, codes, (long)nb * 128, scales, M, nb * BN, kb, act, err, s);
}
