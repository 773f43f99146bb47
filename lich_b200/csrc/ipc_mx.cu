// Storing and reading back microscaled operands (formats and layouts: ipc_mx.cuh).
//
// All four kernels are bound by memory: every input element is read once, every code and scale byte written
// once.  A CTA owns a tile of 32 rows x 256 columns, so that the scale bytes of a tile, which lie across the rows in
// both layouts, leave as whole sectors.
#include "ipc_mx.cuh"

namespace ipc {
namespace {

constexpr int TR = 32;        // rows of a tile
constexpr int TCOL = 256;     // columns of a tile: 8 blocks
constexpr int THREADS = 256;
constexpr int TB = TCOL / MX_BLOCK;

template <typename T>
struct Vec16 {  // 16 consecutive elements
  static __device__ __forceinline__ void load(const T* p, float (&v)[16]) {
    constexpr int N = 16 / sizeof(T);
    uint4 raw[16 / N];
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const T* h = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = St<T>::ld(h[j]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[16]) {
    constexpr int N = 16 / sizeof(T);
    uint4 raw[16 / N];
    T* h = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int j = 0; j < 16; ++j) h[j] = St<T>::st(v[j]);
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
  }
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// f in fp32.  sigmoid and silu take the exponential of -|v|, which cannot overflow: 1 / (1 + e^-v) itself is 0 below
// v = -88.7, where sigmoid(v) is still a (subnormal) number.  Far below 0 silu is v e^v, whose e^v alone would be
// rounded as a subnormal before v multiplies it: the last factor e^-32 is applied at the end.
template <int ACT>
__device__ __forceinline__ float act_full(float v) {
  if constexpr (ACT == IPC_ACT_SIGMOID || ACT == IPC_ACT_SILU) {
    if (ACT == IPC_ACT_SILU && v < -64.f) return v * expf(v + 32.f) * 1.26641655e-14f;
    const float z = expf(-fabsf(v));
    const float n = v >= 0.f ? 1.f : z;
    return (ACT == IPC_ACT_SILU ? v * n : n) / (1.f + z);
  }
  return act_f<ACT>(v);
}
// f of a value that is then stored in T: the MUFU forms for 16-bit storage (their error is about one rounding
// step of fp16), CUDA's own functions for fp32.
template <typename T, int ACT>
__device__ __forceinline__ float act_for(float v) {
  if constexpr (sizeof(T) == 2) return act_f_hw<ACT>(v);
  return act_full<ACT>(v);
}

// ---------------------------------------------------------------------------- 8 bits
// VEC: rows start on 16-byte boundaries; a thread takes 16 elements, two threads a block.  Otherwise a lane
// takes one element of a block, so that loads and stores stay coalesced whatever the row stride.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) mx8_store_kernel(const T* __restrict__ x, signed char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, int D, int B, int nb) {
  __shared__ unsigned char s_scale[TB][TR];
  const int d0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long ldc = (long long)nb * MX_BLOCK;
  if constexpr (VEC) {
    const int cj = tid & 15, r0 = tid >> 4;
#pragma unroll
    for (int it = 0; it < TR / 16; ++it) {
      const int r = r0 + 16 * it, d = d0 + r, c = c0 + 16 * cj;
      float v[16];
      uint32_t m = 0;
      if (d < D && c < B) {
        if (c + 16 <= B) {
          Vec16<T>::load(x + (long long)d * B + c, v);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = c + j < B ? St<T>::ld(x[(long long)d * B + c + j]) : 0.f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, abs_bits(v[j]));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      const uint32_t byte = mx8_scale_byte(m);
      const float inv = mx_inv_scale(byte);
      if ((cj & 1) == 0) s_scale[cj >> 1][r] = (unsigned char)byte;
      if (d < D && c < ldc) {
        uint4 o;
        uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t t = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) t |= ((uint32_t)mx8_code(v[4 * q + j], inv) & 0xffu) << (8 * j);
          w[q] = t;
        }
        *reinterpret_cast<uint4*>(codes + (long long)d * ldc + c) = o;
      }
    }
  } else {
    for (int r = warp; r < TR; r += THREADS / 32) {
      const int d = d0 + r;
      float v[TB];
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int c = c0 + MX_BLOCK * j + lane;
        v[j] = (d < D && c < B) ? St<T>::ld(x[(long long)d * B + c]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const uint32_t byte = mx8_scale_byte(__reduce_max_sync(0xffffffffu, abs_bits(v[j])));
        if (lane == 0) s_scale[j][r] = (unsigned char)byte;
        const int c = c0 + MX_BLOCK * j + lane;
        if (d < D && c < ldc) codes[(long long)d * ldc + c] = (signed char)mx8_code(v[j], mx_inv_scale(byte));
      }
    }
  }
  __syncthreads();
  const int j = c0 / MX_BLOCK + warp;  // eight warps, eight blocks; a lane per row
  if (j < nb && d0 + lane < D) scales[(long long)j * D + d0 + lane] = s_scale[warp][lane];
}

template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(THREADS)
    mx8_restore_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ scales,
                       T* __restrict__ out, int D, int B, int nb, long long ld_out, int pad_cols) {
  const int d0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long ldc = (long long)nb * MX_BLOCK;
  if constexpr (VEC) {
    const int cj = tid & 15, r0 = tid >> 4;
#pragma unroll
    for (int it = 0; it < TR / 16; ++it) {
      const int d = d0 + r0 + 16 * it, c = c0 + 16 * cj;
      if (d >= D || c >= pad_cols) continue;
      float v[16];
      if (c < ldc) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(codes + (long long)d * ldc + c));
        const float sc = mx_scale(scales[(long long)(c / MX_BLOCK) * D + d]);
        const signed char* q = reinterpret_cast<const signed char*>(&raw);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = c + j < B ? act_for<T, ACT>((float)q[j] * sc) : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
      }
      T* o = out + (long long)d * ld_out + c;
      if (c + 16 <= pad_cols) {
        Vec16<T>::store(o, v);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < pad_cols) o[j] = St<T>::st(v[j]);
      }
    }
  } else {
    for (int r = warp; r < TR; r += THREADS / 32) {
      const int d = d0 + r;
      if (d >= D) break;
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int c = c0 + MX_BLOCK * j + lane;
        if (c >= pad_cols) continue;
        float v = 0.f;
        if (c < B)
          v = act_for<T, ACT>((float)codes[(long long)d * ldc + c] *
                              mx_scale(scales[(long long)(c / MX_BLOCK) * D + d]));
        out[(long long)d * ld_out + c] = St<T>::st(v);
      }
    }
  }
}

// ---------------------------------------------------------------------------- 4 bits
// Rows as stored ([R, K], weights): the mapping of mx8_store_kernel, blocks along the row.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(THREADS) mx4_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                           unsigned char* __restrict__ scales, int R, int K, int kp) {
  __shared__ __align__(16) unsigned char s_scale[TR][TB];
  const int r0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x;
  const int cj = tid & 15, rr = tid >> 4;
#pragma unroll
  for (int it = 0; it < TR / 16; ++it) {
    const int r = r0 + rr + 16 * it, c = c0 + 16 * cj;
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.f;
    if (r < R && c < K) {
      if (VEC && c + 16 <= K) {
        Vec16<T>::load(x + (long long)r * K + c, v);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < K) v[j] = St<T>::ld(x[(long long)r * K + c + j]);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = c + j < K ? act_full<ACT>(v[j]) : 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, abs_bits(v[j]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t byte = mx4_scale_byte(m);
    if ((cj & 1) == 0) s_scale[rr + 16 * it][cj >> 1] = (unsigned char)byte;
    if (r < R && c < kp) {
      const float inv = mx_inv_scale(byte);
      float a[8], b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = byte == MX_NAN_BYTE ? 0.f : v[j] * inv;
        b[j] = byte == MX_NAN_BYTE ? 0.f : v[8 + j] * inv;
      }
      *reinterpret_cast<uint2*>(codes + (long long)r * (kp / 2) + c / 2) = make_uint2(mx4_pack8(a), mx4_pack8(b));
    }
  }
  __syncthreads();
  // 32 rows x 2 atoms of 4 blocks: a word each (rows past R belong to the atom's padding and get 0)
  if (tid < 2 * TR) {
    const int r = tid >> 1, a = tid & 1;
    const int j0 = c0 / MX_BLOCK + 4 * a;
    if (j0 * MX_BLOCK < kp)
      *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(r0 + r, j0, kp / 128)) =
          *reinterpret_cast<const uint32_t*>(&s_scale[r][4 * a]);
  }
}

// Turned ([K, R] feature-major states -> R rows of K): a CTA takes 256 features x 64 samples; a warp a block of
// 32 features, a lane two samples, whose 32 values it reads along the samples (coalesced) and keeps in registers.
// The codes pass through shared memory so that a sample's 128 bytes leave together.
constexpr int TUR = 64;
template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS) mx4_turned_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, int R, int K, int kp) {
  __shared__ __align__(16) unsigned char s_code[TUR][144];  // 128 bytes of codes per sample, rows 16 bytes apart mod 128
  __shared__ __align__(16) unsigned char s_scale[TUR][TB];
  const int r0 = blockIdx.x * TUR, k0 = blockIdx.y * TCOL;  // neighbouring CTAs read neighbouring samples
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kb = k0 + MX_BLOCK * warp;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + 32 * h + lane;
    float v[MX_BLOCK];
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i)
      v[i] = (r < R && kb + i < K) ? St<T>::ld(x[(long long)(kb + i) * R + r]) : 0.f;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i) {
      v[i] = (r < R && kb + i < K) ? act_full<ACT>(v[i]) : 0.f;
      m = max(m, abs_bits(v[i]));
    }
    const uint32_t byte = mx4_scale_byte(m);
    const float inv = mx_inv_scale(byte);
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float a[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = byte == MX_NAN_BYTE ? 0.f : v[8 * q + j] * inv;
      w[q] = mx4_pack8(a);
    }
    *reinterpret_cast<uint4*>(&s_code[32 * h + lane][16 * warp]) = o;
    s_scale[32 * h + lane][warp] = (unsigned char)byte;
  }
  __syncthreads();
#pragma unroll
  for (int i = tid; i < TUR * 8; i += THREADS) {
    const int r = i >> 3, c = i & 7;
    if (r0 + r < R && k0 + 32 * c < kp)
      *reinterpret_cast<uint4*>(codes + (long long)(r0 + r) * (kp / 2) + k0 / 2 + 16 * c) =
          *reinterpret_cast<const uint4*>(&s_code[r][16 * c]);
  }
  if (tid < 2 * TUR) {
    const int r = tid >> 1, a = tid & 1;
    const int j0 = k0 / MX_BLOCK + 4 * a;
    if (j0 * MX_BLOCK < kp)
      *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(r0 + r, j0, kp / 128)) =
          *reinterpret_cast<const uint32_t*>(&s_scale[r][4 * a]);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) mx4_restore_kernel(const unsigned char* __restrict__ codes,
                                                              const unsigned char* __restrict__ scales,
                                                              T* __restrict__ out, int R, int K, int kp) {
  const int r0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x;
  const int cj = tid & 15, rr = tid >> 4;
#pragma unroll
  for (int it = 0; it < TR / 16; ++it) {
    const int r = r0 + rr + 16 * it, c = c0 + 16 * cj;
    if (r >= R || c >= K) continue;
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + (long long)r * (kp / 2) + c / 2));
    const float sc = mx_scale(scales[mx4_scale_at(r, c / MX_BLOCK, kp / 128)]);
    uint32_t h[8];
    mx4_unpack8(q.x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
    mx4_unpack8(q.y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
    float v[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      v[2 * j] = f.x * sc;
      v[2 * j + 1] = f.y * sc;
    }
    T* o = out + (long long)r * K + c;
    if (VEC && c + 16 <= K) {
      Vec16<T>::store(o, v);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c + j < K) o[j] = St<T>::st(v[j]);
    }
  }
}

template <typename T>
bool rows_aligned(const void* p, long long ld) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (long long)sizeof(T))) & 15) == 0;
}

int grid_of(const char* what, long long rows, int tile, long long cols, dim3* grid) {
  const long long gy = (rows + tile - 1) / tile, gx = (cols + TCOL - 1) / TCOL;
  if (gy > 65535 || gx > 0x7fffffffLL) return set_error(IPC_ERR_ARG, "%s: %lld rows are too many", what, rows);
  *grid = dim3((unsigned)gx, (unsigned)gy);
  return IPC_OK;
}

}  // namespace

int launch_mx8_store(const void* x, signed char* codes, unsigned char* scales, int D, int B, int dtype, cudaStream_t s) {
  const int nb = (int)(mx8_ld(B) / MX_BLOCK);
  dim3 grid;
  int rc = grid_of("8-bit store", D, TR, B, &grid);
  if (rc) return rc;
  IPC_DISPATCH_DT(dtype, TT, {
    const TT* xt = static_cast<const TT*>(x);
    if (rows_aligned<TT>(x, B))
      mx8_store_kernel<TT, true><<<grid, THREADS, 0, s>>>(xt, codes, scales, D, B, nb);
    else
      mx8_store_kernel<TT, false><<<grid, THREADS, 0, s>>>(xt, codes, scales, D, B, nb);
  });
  count_launch();
  return check_launch("8-bit store");
}

int launch_mx8_restore(const signed char* codes, const unsigned char* scales, void* out, int D, int B, long long ld_out,
                       int pad_cols, int act, int dtype, cudaStream_t s) {
  const int nb = (int)(mx8_ld(B) / MX_BLOCK);
  dim3 grid;
  int rc = grid_of("8-bit restore", D, TR, pad_cols, &grid);
  if (rc) return rc;
  IPC_DISPATCH_DT(dtype, TT, {
    TT* ot = static_cast<TT*>(out);
    const bool vec = rows_aligned<TT>(out, ld_out);
    IPC_DISPATCH_ACT(act, AC, {
      if (vec)
        mx8_restore_kernel<TT, AC, true><<<grid, THREADS, 0, s>>>(codes, scales, ot, D, B, nb, ld_out, pad_cols);
      else
        mx8_restore_kernel<TT, AC, false><<<grid, THREADS, 0, s>>>(codes, scales, ot, D, B, nb, ld_out, pad_cols);
    });
  });
  count_launch();
  return check_launch("8-bit restore");
}

int launch_mx4_quantize(const void* x, unsigned char* codes, unsigned char* scales, int R, int K, int turned, int act,
                        int dtype, cudaStream_t s) {
  const int kp = (int)mx4_kp(K);
  if (turned && (kp + TCOL - 1) / TCOL > 65535) return set_error(IPC_ERR_ARG, "4-bit quantisation: K=%d is too large", K);
  const long long rows = ((long long)R + 127) / 128 * 128;  // the scale atoms' padding rows are written too
  dim3 grid;
  int rc = IPC_OK;
  if (turned)
    grid = dim3((unsigned)(rows / TUR), (unsigned)((kp + TCOL - 1) / TCOL));
  else
    rc = grid_of("4-bit quantisation", rows, TR, kp, &grid);
  if (rc) return rc;
  IPC_DISPATCH_DT(dtype, TT, {
    const TT* xt = static_cast<const TT*>(x);
    const bool vec = rows_aligned<TT>(x, K);
    IPC_DISPATCH_ACT(act, AC, {
      if (turned)
        mx4_turned_kernel<TT, AC><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
      else if (vec)
        mx4_rows_kernel<TT, AC, true><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
      else
        mx4_rows_kernel<TT, AC, false><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
    });
  });
  count_launch();
  return check_launch("4-bit quantisation");
}

int launch_mx4_restore(const unsigned char* codes, const unsigned char* scales, void* out, int R, int K, int dtype,
                       cudaStream_t s) {
  const int kp = (int)mx4_kp(K);
  dim3 grid;
  int rc = grid_of("4-bit restore", R, TR, K, &grid);
  if (rc) return rc;
  IPC_DISPATCH_DT(dtype, TT, {
    TT* ot = static_cast<TT*>(out);
    if (rows_aligned<TT>(out, K))
      mx4_restore_kernel<TT, true><<<grid, THREADS, 0, s>>>(codes, scales, ot, R, K, kp);
    else
      mx4_restore_kernel<TT, false><<<grid, THREADS, 0, s>>>(codes, scales, ot, R, K, kp);
  });
  count_launch();
  return check_launch("4-bit restore");
}

}  // namespace ipc
