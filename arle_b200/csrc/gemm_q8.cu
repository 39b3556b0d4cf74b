// Products of e4m3 codes with a scale for each block of 128 numbers of k:
//     out[m, n] = sum over blocks b of  sx[m, b] * sw[n / 128, b] * sum over k in b of  x[m, k] * w[n, k]
// x [M, K] and w [N, K] codes, K = 128 kb (filled up with codes of zero), sx powers of two (one byte: exponent + 127), sw float32.  A block's inner sum is
// formed by the tensor cores in float32 (products of two codes are exact), every block's sum is scaled by sx sw and added up in float32, in the order of k and then of
// the warps or parts that shared k: (127 + kb + 2) half steps of the terms' magnitudes at most.  The store rounds to bfloat16 or not at all.
#include "q8.cuh"
using namespace arle;

namespace {

constexpr int kBlock = 128;

// c += a . b on codes: a 16 x 32 (rows g and g + 8, bytes 4t.. and 16 + 4t..), b 32 x 8 (column g), c as for bfloat16; g = lane / 4, t = lane % 4.
__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A plain load of what is read once, which stays behind pdl_wait.
__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Few rows: bound by the bytes of w, read straight from memory into the operands of mma.sync.  A block owns 16 rows of w and up to eight rows of x; its warp i
// takes the blocks i, i + WARPS, ... of k.  The order of k inside a block of 128 is free as long as both operands have the same: lane (g, t) takes bytes
// 32t .. 32t + 31 of its row's block, so a warp's loads cover whole 128-byte lines, and words 2i and 2i + 1 of those are the operands of the i-th of
// four mma.  What hides the memory is many warps, a block of k each on its way, not several blocks in a warp: with two, and with rings of four that go on
// across rows, all sizes took longer (4,096 x 12,288 for one row 15 to 26 us instead of 10.3), and so did x fetched a block ahead.
// A warp has the block of k behind the next one brought to L2 meanwhile: in decode steps of 14 layers of 8B sizes, 193 MB each, a layer takes 53.6 us for 56.0 (one
// request; the products by themselves gain 0 to 3 %, as weights in turn of 2 GB; everything a warp has left brought at once, or by bulk copies, takes 3 to 7 us more).
// The first two blocks of w of every warp are brought to L2 while the kernel in front ends and read behind the wait for it, since it may have written them (read in front
// of it: 5.1 us for 5.3, one row of 4,096 x 4,096; a layer of 8B sizes for one request 54.2 for 55.3).  The next kernel may start when a block's sums are done and not
// before: long blocks that start early gather on the SMs that have room (the decode attention of eight requests behind a product, and so a layer of 8B sizes, took
// 20 us more: 81 and 61), and short ones gain nothing (norms, codes and the four products of a layer for one row 46.1 and 44.8 us).
// One row, us and TB/s, weights in turn of 2 GB: 4,096 x 4,096 5.3 (3.1), 4,096 x 12,288 10.4 (4.8), 6,144 x 4,096 6.4 (3.9), 24,576 x 4,096 18.5 (5.4); eight
// rows some 3 % more.
template <int WARPS, int BLOCKS, typename OutT>
__global__ void __launch_bounds__(32 * WARPS, BLOCKS) gemm_q8_rows_kernel(const uint8_t* x, const uint8_t* sx, const uint8_t* w, const float* sw, OutT* out, long ldo,
                                                                         int M, int N, int kb) {
  __shared__ float part[WARPS][16][9];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8;
  const size_t K = (size_t)kb * kBlock;
  const uint8_t* w0 = w + (size_t)min(n0 + g, N - 1) * K + 32 * t;
  const uint8_t* w1 = w + (size_t)min(n0 + g + 8, N - 1) * K + 32 * t;
  const float* swr = sw + (size_t)(n0 / kBlock) * kb;
  uint4 a[4];
  auto ask = [&](int b) {
    if (b < kb) {
      const size_t at = (size_t)b * kBlock;
      a[0] = load_once(w0 + at), a[1] = load_once(w0 + at + 16), a[2] = load_once(w1 + at), a[3] = load_once(w1 + at + 16);
    }
  };
  auto hint = [&](int b) {                                 // a row's block of k is one line
    if (t == 0 && b < kb) {
      asm volatile("prefetch.global.L2 [%0];\n" ::"l"(w0 + (size_t)b * kBlock) : "memory");
      asm volatile("prefetch.global.L2 [%0];\n" ::"l"(w1 + (size_t)b * kBlock) : "memory");
    }
  };
  hint(warp);
  hint(warp + WARPS);
  pdl_wait();
  ask(warp);
  const uint8_t* xr = x + (size_t)min(m0 + g, M - 1) * K + 32 * t;
  const uint8_t* sxa = sx + (size_t)min(m0 + 2 * t, M - 1) * kb;
  const uint8_t* sxb = sx + (size_t)min(m0 + 2 * t + 1, M - 1) * kb;
  float acc[4] = {};
  for (int b = warp; b < kb; b += WARPS) {
    const uint4 x0 = *reinterpret_cast<const uint4*>(xr + (size_t)b * kBlock), x1 = *reinterpret_cast<const uint4*>(xr + (size_t)b * kBlock + 16);
    const float s = swr[b], fa = s * __uint_as_float((uint32_t)sxa[b] << 23), fb = s * __uint_as_float((uint32_t)sxb[b] << 23);
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    mma_e4m3(d, a[0].x, a[2].x, a[0].y, a[2].y, x0.x, x0.y);
    mma_e4m3(d, a[0].z, a[2].z, a[0].w, a[2].w, x0.z, x0.w);
    mma_e4m3(d, a[1].x, a[3].x, a[1].y, a[3].y, x1.x, x1.y);
    mma_e4m3(d, a[1].z, a[3].z, a[1].w, a[3].w, x1.z, x1.w);
    acc[0] = fmaf(d[0], fa, acc[0]), acc[1] = fmaf(d[1], fb, acc[1]);
    acc[2] = fmaf(d[2], fa, acc[2]), acc[3] = fmaf(d[3], fb, acc[3]);
    hint(b + 2 * WARPS);
    ask(b + WARPS);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][2 * t + (e & 1)] = acc[e];
  __syncthreads();
  pdl_launch_dependents();
  if (threadIdx.x < 128) {                                 // added up in the order of the warps
    const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) v += part[k][n][m];
    if (n0 + n < N && m0 + m < M) out[(size_t)(m0 + m) * ldo + n0 + n] = from_f32<OutT>(v);
  }
}

template <typename OutT>
int product(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, cudaStream_t s) {
  const int tiles = (N + 15) / 16, tiles_m = (M + 7) / 8;
  if (tiles_m > 65535) return ARLE_E_UNSUPPORTED;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // 16 warps to a tile where all tiles are under way at once, else eight: us for one row behind the launch of its codes with 16 warps, eight in three blocks an SM and
  // eight in four, 4,096 x 12,288 (256 tiles) 11.4, 12.1 and 13.0; 6,144 x 4,096 (384) 8.6, 7.1 and 7.4; 24,576 x 4,096 (1,536) 21.5, 20.0 and 19.4
  const long blocks = (long)tiles * tiles_m;
  const int warps = blocks <= 2l * sms ? 16 : 8;
  auto kern = blocks <= 2l * sms ? gemm_q8_rows_kernel<16, 2, OutT> : blocks <= 3l * sms ? gemm_q8_rows_kernel<8, 3, OutT> : gemm_q8_rows_kernel<8, 4, OutT>;
  launch_early(kern, dim3(tiles, tiles_m), dim3(32 * warps), 0, s, 1, (const uint8_t*)x, (const uint8_t*)sx, (const uint8_t*)w, sw, (OutT*)out, ldo, M, N, kb);
  return launch_status();
}

}  // namespace

// x [M, 128 kb], sx [M, kb], w [N, 128 kb] (both on 16-byte boundaries), sw [ceil(N / 128), kb], out [M, N] of rows ldo apart (0 float32, 1 bfloat16).
ARLE_API int arle_gemm_q8(const void* x, const void* sx, const void* w, const float* sw, void* out, int out_dtype, long ldo, int M, int N, int kb,
                          cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (kb <= 0 || (((uintptr_t)x | (uintptr_t)w) & 15)) return ARLE_E_BADARG;
  if (out_dtype == 0) return product<float>(x, sx, w, sw, out, ldo, M, N, kb, s);
  if (out_dtype == 1) return product<__nv_bfloat16>(x, sx, w, sw, out, ldo, M, N, kb, s);
  return ARLE_E_BADARG;
}
