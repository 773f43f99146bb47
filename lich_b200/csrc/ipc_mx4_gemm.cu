// out [M, B] = W4 [M, K] @ A4 [B, K]^T for 4-bit operands in blocks of 32 along K (ipc_mx.cuh).
//
// The plain form of the product: tiles of 64 x 64, both operands read back to bf16 in shared memory (c * 2^s is exact
// there) and multiplied with mma.sync, fp32 accumulators.
#include "ipc_mx.cuh"

namespace ipc {
namespace {

constexpr int PT = 64, PK = 128, PLD = PK + 8, PTHREADS = 128;

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// 64 rows x 128 columns of an operand -> bf16; a thread reads 32 bytes (two blocks) of a row
__device__ __forceinline__ void stage(__nv_bfloat16 (*dst)[PLD], const unsigned char* codes, const unsigned char* scales,
                                      int rows, int r0, int k0, int kp) {
  const int r = threadIdx.x >> 1, half = threadIdx.x & 1;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int k = k0 + 64 * half + 32 * b;
    uint4 q = make_uint4(0, 0, 0, 0);
    float sc = 0.f;
    if (r0 + r < rows) {
      q = __ldg(reinterpret_cast<const uint4*>(codes + (long long)(r0 + r) * (kp / 2) + k / 2));
      sc = mx_scale(scales[mx4_scale_at(r0 + r, k / MX_BLOCK, kp / 128)]);
    }
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h[4];
      mx4_unpack8(w[i], h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        *reinterpret_cast<__nv_bfloat162*>(&dst[r][64 * half + 32 * b + 8 * i + 2 * j]) =
            __floats2bfloat162_rn(f.x * sc, f.y * sc);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(PTHREADS)
    mx4_plain_gemm_kernel(const unsigned char* __restrict__ w, const unsigned char* __restrict__ wsc,
                          const unsigned char* __restrict__ a, const unsigned char* __restrict__ asc,
                          T* __restrict__ out, int M, int B, int kp) {
  __shared__ __align__(16) __nv_bfloat16 sW[PT][PLD];
  __shared__ __align__(16) __nv_bfloat16 sA[PT][PLD];
  const int m0 = blockIdx.y * PT, n0 = blockIdx.x * PT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp >> 1, wn = warp & 1, gq = lane >> 2, tq = lane & 3;
  float acc[2][4][4] = {};
  for (int k0 = 0; k0 < kp; k0 += PK) {
    stage(sW, w, wsc, M, m0, k0, kp);
    stage(sA, a, asc, B, n0, k0, kp);
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < PK; ks += 16) {
      uint32_t fa[2][4], fb[4][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = wm * 32 + i * 16 + gq;
        fa[i][0] = *reinterpret_cast<const uint32_t*>(&sW[r][ks + 2 * tq]);
        fa[i][1] = *reinterpret_cast<const uint32_t*>(&sW[r + 8][ks + 2 * tq]);
        fa[i][2] = *reinterpret_cast<const uint32_t*>(&sW[r][ks + 2 * tq + 8]);
        fa[i][3] = *reinterpret_cast<const uint32_t*>(&sW[r + 8][ks + 2 * tq + 8]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = wn * 32 + j * 8 + gq;
        fb[j][0] = *reinterpret_cast<const uint32_t*>(&sA[c][ks + 2 * tq]);
        fb[j][1] = *reinterpret_cast<const uint32_t*>(&sA[c][ks + 2 * tq + 8]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_bf16(acc[i][j], fa[i], fb[j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + wm * 32 + i * 16 + gq + (r >= 2 ? 8 : 0);
        const int n = n0 + wn * 32 + j * 8 + 2 * tq + (r & 1);
        if (m < M && n < B) out[(long long)m * B + n] = St<T>::st(acc[i][j][r]);
      }
}

}  // namespace

int launch_mx4_gemm(const unsigned char* w, const unsigned char* wsc, const unsigned char* a, const unsigned char* asc,
                    void* out, int M, int K, int B, int dtype, cudaStream_t s) {
  const int kp = (int)mx4_kp(K);
  const dim3 grid((unsigned)((B + PT - 1) / PT), (unsigned)((M + PT - 1) / PT));
  if (grid.y > 65535u) return set_error(IPC_ERR_ARG, "4-bit product: M=%d is too large", M);
  IPC_DISPATCH_DT(dtype, TT, {
    mx4_plain_gemm_kernel<TT><<<grid, PTHREADS, 0, s>>>(w, wsc, a, asc, static_cast<TT*>(out), M, B, kp);
  });
  count_launch();
  return check_launch("4-bit product");
}

}  // namespace ipc
