// Products of e4m3 codes with a scale for each block of 128 numbers of k:
//     out[m, n] = sum over blocks b of  sx[m, b] * sw[n / 128, b] * sum over k in b of  x[m, k] * w[n, k]
// x [M, K] and w [N, K] codes, K = 128 kb (filled up with codes of zero), sx powers of two (one byte: exponent + 127), sw float32.  A block's inner sum is
// formed by the tensor cores, every block's sum is scaled and added up in float32 registers; the only rounding is the store (bfloat16 or none).
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

// A block of eight warps owns 16 rows of w and up to 8 MT rows of x; warp i takes the blocks i, i + 8, ... of k.  The order of k inside a block of 128 is
// free as long as both operands have the same: lane (g, t) takes bytes 32t .. 32t + 31 of its row's block, so a warp's loads cover whole 128-byte lines,
// and words 2i and 2i + 1 of those are the operands of the i-th of four mma.
template <int MT, typename OutT>
__global__ void __launch_bounds__(256) gemm_q8_rows_kernel(const uint8_t* x, const uint8_t* sx, const uint8_t* w, const float* sw, OutT* out, long ldo, int M,
                                                           int N, int kb) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int TOKENS = 8 * MT;
  __shared__ float part[8][16][TOKENS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * TOKENS;
  const size_t K = (size_t)kb * kBlock;
  const uint8_t* wr[2] = {w + min(n0 + g, N - 1) * K + 32 * t, w + min(n0 + g + 8, N - 1) * K + 32 * t};
  const float* swr = sw + (size_t)(n0 / kBlock) * kb;
  float acc[MT][4] = {};
  for (int b = warp; b < kb; b += 8) {
    uint4 a[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) a[r][h] = *reinterpret_cast<const uint4*>(wr[r] + (size_t)b * kBlock + 16 * h);
    const float s = swr[b];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const uint8_t* xr = x + min(m0 + 8 * j + g, M - 1) * K + (size_t)b * kBlock + 32 * t;
      const uint4 x0 = *reinterpret_cast<const uint4*>(xr), x1 = *reinterpret_cast<const uint4*>(xr + 16);
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      mma_e4m3(d, a[0][0].x, a[1][0].x, a[0][0].y, a[1][0].y, x0.x, x0.y);
      mma_e4m3(d, a[0][0].z, a[1][0].z, a[0][0].w, a[1][0].w, x0.z, x0.w);
      mma_e4m3(d, a[0][1].x, a[1][1].x, a[0][1].y, a[1][1].y, x1.x, x1.y);
      mma_e4m3(d, a[0][1].z, a[1][1].z, a[0][1].w, a[1][1].w, x1.z, x1.w);
      const int ma = min(m0 + 8 * j + 2 * t, M - 1), mb = min(m0 + 8 * j + 2 * t + 1, M - 1);
      const float fa = s * __uint_as_float((uint32_t)sx[(size_t)ma * kb + b] << 23), fb = s * __uint_as_float((uint32_t)sx[(size_t)mb * kb + b] << 23);
      acc[j][0] = fmaf(d[0], fa, acc[j][0]), acc[j][1] = fmaf(d[1], fb, acc[j][1]);
      acc[j][2] = fmaf(d[2], fa, acc[j][2]), acc[j][3] = fmaf(d[3], fb, acc[j][3]);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][8 * j + 2 * t + (e & 1)] = acc[j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * TOKENS; i += 256) {
    const int n = i & 15, m = i >> 4;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += part[k][n][m];
    if (n0 + n < N && m0 + m < M) out[(size_t)(m0 + m) * ldo + n0 + n] = from_f32<OutT>(v);
  }
}

template <int MT, typename OutT>
int launch_rows(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, cudaStream_t s) {
  const int tiles_m = (M + 8 * MT - 1) / (8 * MT);
  if (tiles_m > 65535) return ARLE_E_UNSUPPORTED;
  launch_kernel(gemm_q8_rows_kernel<MT, OutT>, dim3((N + 15) / 16, tiles_m), dim3(256), 0, s, 1, (const uint8_t*)x, (const uint8_t*)sx, (const uint8_t*)w, sw,
                (OutT*)out, ldo, M, N, kb);
  return launch_status();
}

template <typename OutT>
int product(const void* x, const void* sx, const void* w, const float* sw, void* out, long ldo, int M, int N, int kb, cudaStream_t s) {
  if (M <= 8) return launch_rows<1, OutT>(x, sx, w, sw, out, ldo, M, N, kb, s);
  return launch_rows<4, OutT>(x, sx, w, sw, out, ldo, M, N, kb, s);
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
