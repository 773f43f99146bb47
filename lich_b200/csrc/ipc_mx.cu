// Storing and reading back microscaled operands (formats and layouts: ipc_mx.cuh).
//
// These kernels are bound by memory: every input element is read once, every code and scale byte written once.  A CTA
// owns a tile of 32 rows x 256 columns, so that the scale bytes of a tile, which lie across the rows in both layouts,
// leave as whole sectors.  A thread that restores writes one 16-byte vector at a time, so that a warp instruction covers
// whole sectors (with two vectors a thread the stores reach L2 as half sectors: 22 us against 17 us for 8-bit codes at
// 4096 x 8192 in bf16).  Rows that do not start on 16-byte boundaries take a lane per element.
#include "ipc_mx.cuh"
#include "ipc_ptx.cuh"

namespace ipc {
namespace {

constexpr int TR = 32;        // rows of a tile
constexpr int TCOL = 256;     // columns of a tile: 8 blocks
constexpr int THREADS = 256;
// A lane per element: up to a warp per row of the tile, so that small odd matrices need one round of loads (1000 x 777: 5 us a
// kernel with 256 threads, 3.3 with 1024).  The 8-bit kernels keep 256 where tiles fill the GPU anyway (4095 x 4095: 22 us
// against 25 and 29; the 4-bit ones, whose loads are all in registers, 34 and 38 against 27 and 36).
constexpr int LANE_THREADS = 1024;
__host__ __device__ constexpr int threads_of(bool vec) { return vec ? THREADS : LANE_THREADS; }
constexpr int TB = TCOL / MX_BLOCK;

template <typename T>
struct Vec {  // one 16-byte vector
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void load(const T* p, float (&v)[N]) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = St<T>::ld(h[j]);
  }
  // bits (of a float) of the largest magnitude.  16-bit types: compared as they are, two at a time; the bits of a
  // magnitude grow with it in either type, and a NaN's lie above infinity's.
  static __device__ __forceinline__ uint32_t max_bits(const uint4& raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) {
      return max(max(w[0] & 0x7fffffffu, w[1] & 0x7fffffffu), max(w[2] & 0x7fffffffu, w[3] & 0x7fffffffu));
    } else {
      const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                  __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
      const uint16_t b = (uint16_t)max(m & 0xffffu, m >> 16);
      return __float_as_uint(St<T>::ld(*reinterpret_cast<const T*>(&b)));
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    uint4 raw;
    T* h = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = St<T>::st(v[j]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
};
// N codes (bytes) moved at once
__device__ __forceinline__ void ld_codes(const void* p, uint32_t (&w)[2]) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
  w[0] = v.x; w[1] = v.y;
}
__device__ __forceinline__ void ld_codes(const void* p, uint32_t (&w)[1]) { w[0] = __ldg(reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ void st_codes(void* p, const uint32_t (&w)[2]) { *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void st_codes(void* p, const uint32_t (&w)[4]) { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void st_codes(void* p, const uint32_t (&w)[1]) { *reinterpret_cast<uint32_t*>(p) = w[0]; }
// the largest of a block's magnitudes, the block spread over G neighbouring lanes
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
  for (int o = 1; o < G; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// ... of f(x): relu leaves no sign bit (nor does the NaN that max.NaN gives)
template <int ACT>
__device__ __forceinline__ uint32_t f_bits(float v) {
  return ACT == IPC_ACT_RELU ? __float_as_uint(v) : abs_bits(v);
}

// words of a later kernel's workspace, cleared by the first CTA
__device__ __forceinline__ void zero_words(int* zero, int n) {
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < n; i += THREADS) zero[i] = 0;
}

// ---------------------------------------------------------------------------- 8 bits
// VEC: rows start on 16-byte boundaries (so B is a multiple of a vector); 2 threads a block (8 in fp32): the kernel is bound by
// the instructions it issues, and 16 numbers a thread share a magnitude, a scale and two addresses.
template <typename T, bool VEC>
__global__ void __launch_bounds__(threads_of(VEC)) mx8_store_kernel(const T* __restrict__ x, signed char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, int D, int B, int nb) {
  __shared__ unsigned char s_scale[TB][TR];
  const int d0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long ldc = (long long)nb * MX_BLOCK;
  if constexpr (VEC) {
    constexpr int V = Vec<T>::N, NV = sizeof(T) == 2 ? 2 : 1, N = V * NV;  // vectors and numbers of a thread
    constexpr int TPR = TCOL / N, RPI = THREADS / TPR;                     // threads a row, rows at a time
    const int c = c0 + N * (tid % TPR);
    uint4 raw[TR / RPI][NV];
#pragma unroll
    for (int it = 0; it < TR / RPI; ++it) {  // all loads first
      const int d = d0 + tid / TPR + RPI * it;
#pragma unroll
      for (int h = 0; h < NV; ++h) {
        raw[it][h] = make_uint4(0, 0, 0, 0);
        if (d < D && c + V * h < B) raw[it][h] = __ldg(reinterpret_cast<const uint4*>(x + (long long)d * B + c) + h);
      }
    }
#pragma unroll
    for (int it = 0; it < TR / RPI; ++it) {
      const int r = tid / TPR + RPI * it, d = d0 + r;
      uint32_t m = Vec<T>::max_bits(raw[it][0]);
      if constexpr (NV == 2) m = max(m, Vec<T>::max_bits(raw[it][1]));
      const uint32_t byte = mx8_scale_byte(group_max<MX_BLOCK / N>(m));
      const float inv = mx_inv_scale(byte);
      if (c % MX_BLOCK == 0) s_scale[(c - c0) / MX_BLOCK][r] = (unsigned char)byte;
      if (d < D && c < ldc) {
        const T* h = reinterpret_cast<const T*>(raw[it]);
        uint32_t w[N / 4];
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
          // v * 2^-s + 1.5 * 2^23: the integer nearest to v * 2^-s (ties to even) in the sum's low byte
          uint32_t t[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = __float_as_uint(fmaf(St<T>::ld(h[4 * q + j]), inv, 12582912.f));
          w[q] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
        }
        if (byte == MX_NAN_BYTE)
#pragma unroll
          for (int q = 0; q < N / 4; ++q) w[q] = 0;
        st_codes(codes + (long long)d * ldc + c, w);
      }
    }
  } else {
    for (int r = warp; r < TR; r += (int)blockDim.x / 32) {
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
  const int j = c0 / MX_BLOCK + warp;  // a warp per block, a lane per row
  if (warp < TB && j < nb && d0 + lane < D) scales[(long long)j * D + d0 + lane] = s_scale[warp][lane];
}

template <typename T, int ACT, bool VEC>
__device__ __forceinline__ void restore_tile(const signed char* __restrict__ codes,
                                             const unsigned char* __restrict__ scales, T* __restrict__ out, int D,
                                             int cols, int nb, long long ld_out) {
  const int d0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long ldc = (long long)nb * MX_BLOCK;
  if constexpr (VEC) {
    constexpr int N = Vec<T>::N, TPR = TCOL / N, RPI = THREADS / TPR, IT = TR / RPI;
    const int c = c0 + N * (tid % TPR);
    if (c >= cols) return;
    uint32_t w[IT][N / 4], byte[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {  // all loads first
      const int d = d0 + tid / TPR + RPI * it;
      byte[it] = 0;
#pragma unroll
      for (int q = 0; q < N / 4; ++q) w[it][q] = 0;
      if (d < D) {
        ld_codes(codes + (long long)d * ldc + c, w[it]);
        byte[it] = __ldg(scales + (long long)(c / MX_BLOCK) * D + d);
      }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int d = d0 + tid / TPR + RPI * it;
      if (d >= D) continue;
      const float sc = mx_scale(byte[it]);
      float v[N];
#pragma unroll
      for (int q = 0; q < N / 4; ++q) mx8_floats(w[it][q], v + 4 * q);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = mx_f<T, ACT>(v[j] * sc);
      T* o = out + (long long)d * ld_out + c;
      if (c + N <= cols) {
        Vec<T>::store(o, v);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (c + j < cols) o[j] = St<T>::st(v[j]);
      }
    }
  } else {
    for (int r = warp; r < TR; r += (int)blockDim.x / 32) {
      const int d = d0 + r;
      if (d >= D) break;
      int q[TB];
      uint32_t byte[TB];
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int c = c0 + MX_BLOCK * j + lane;
        q[j] = c < cols ? __ldg(codes + (long long)d * ldc + c) : 0;
        byte[j] = c < cols ? __ldg(scales + (long long)(c / MX_BLOCK) * D + d) : 0u;
      }
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int c = c0 + MX_BLOCK * j + lane;
        if (c < cols) out[(long long)d * ld_out + c] = St<T>::st(mx_f<T, ACT>((float)q[j] * mx_scale(byte[j])));
      }
    }
  }
}

template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(threads_of(VEC))
    mx8_restore_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ scales,
                       T* __restrict__ out, int D, int cols, int nb, long long ld_out, int* zero, int n_zero) {
  grid_let_next_start();
  zero_words(zero, n_zero);
  restore_tile<T, ACT, VEC>(codes, scales, out, D, cols, nb, ld_out);
}

// ---------------------------------------------------------------------------- 4 bits
// Rows as stored ([R, K], weights): the mapping of mx8_store_kernel, blocks along the row.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(threads_of(VEC)) mx4_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                           unsigned char* __restrict__ scales, int R, int K, int kp) {
  __shared__ __align__(16) unsigned char s_scale[TR][TB];
  const int r0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if constexpr (VEC) {
    constexpr int N = 8, TPR = TCOL / N, RPI = THREADS / TPR;  // 8 codes: 4 bytes a thread
    const int c = c0 + N * (tid % TPR);
    constexpr int NV = N / Vec<T>::N;
    uint4 raw[TR / RPI][NV];
#pragma unroll
    for (int it = 0; it < TR / RPI; ++it)  // all loads first (K is a multiple of a vector)
#pragma unroll
      for (int h = 0; h < NV; ++h) {
        const int r = r0 + tid / TPR + RPI * it, ch = c + h * Vec<T>::N;
        raw[it][h] = make_uint4(0, 0, 0, 0);
        if (r < R && ch < K) raw[it][h] = __ldg(reinterpret_cast<const uint4*>(x + (long long)r * K + ch));
      }
#pragma unroll
    for (int it = 0; it < TR / RPI; ++it) {
      const int rr = tid / TPR + RPI * it, r = r0 + rr;
      float v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const T* h = reinterpret_cast<const T*>(raw[it]);
        v[j] = mx_f<float, ACT>(St<T>::ld(h[j]));
        if (ACT == IPC_ACT_SIGMOID && !(r < R && c + j < K)) v[j] = 0.f;  // (the other f are 0 at 0)
      }
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) m = max(m, f_bits<ACT>(v[j]));
      const uint32_t byte = mx4_scale_byte(group_max<MX_BLOCK / N>(m));
      if (c % MX_BLOCK == 0) s_scale[rr][(c - c0) / MX_BLOCK] = (unsigned char)byte;
      if (r < R && c < kp) {
        const float inv = mx_inv_scale(byte);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = byte == MX_NAN_BYTE ? 0.f : v[j] * inv;
        *reinterpret_cast<uint32_t*>(codes + (long long)r * (kp / 2) + c / 2) = mx4_pack8(v);
      }
    }
  } else {
    constexpr int RW = TR / (LANE_THREADS / 32);  // rows of a warp, all loads first
    float in[RW][TB];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int r = r0 + warp + LANE_THREADS / 32 * i, c = c0 + MX_BLOCK * j + lane;
        in[i][j] = (r < R && c < K) ? St<T>::ld(x[(long long)r * K + c]) : 0.f;
      }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int rr = warp + LANE_THREADS / 32 * i, r = r0 + rr;
      float (&v)[TB] = in[i];
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int c = c0 + MX_BLOCK * j + lane;
        if (ACT != IPC_ACT_RELU && ACT != IPC_ACT_IDENTITY) v[j] = (r < R && c < K) ? mx_f<float, ACT>(v[j]) : 0.f;
        else v[j] = mx_f<float, ACT>(v[j]);
        const uint32_t byte = mx4_scale_byte(__reduce_max_sync(0xffffffffu, f_bits<ACT>(v[j])));
        if (lane == 0) s_scale[rr][j] = (unsigned char)byte;
        const float lo = byte == MX_NAN_BYTE ? 0.f : v[j] * mx_inv_scale(byte);
        const float hi = __shfl_down_sync(0xffffffffu, lo, 1);
        if ((lane & 1) == 0 && r < R && c < kp)
          codes[(long long)r * (kp / 2) + c / 2] = (unsigned char)mx4_pack2(lo, hi);
      }
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
// 32 features, a lane two samples, whose 32 values it reads along the samples (a warp instruction takes 128 bytes of a
// feature) and keeps in registers, so that a block's magnitude and codes need no exchange.  The codes pass through
// shared memory, so that a sample's 128 bytes leave together.
// PAIR: rows start on boundaries of two elements and a lane takes two neighbouring samples; otherwise samples lane, lane + 32.
constexpr int TUR = 64;
// relu of two 16-bit numbers (a NaN stays one)
template <typename T>
__device__ __forceinline__ uint32_t relu2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&w), __float2half2_rn(0.f));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&w), __float2bfloat162_rn(0.f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  return w;
}
template <typename T, bool PAIR>
struct alignas(2 * sizeof(T)) Two {  // an element of each of a lane's two samples
  T v[2];
};
template <typename T, bool PAIR>
__device__ __forceinline__ Two<T, PAIR> load_two(const T* row, int lane, bool in0, bool in1) {
  Two<T, PAIR> t;
  if constexpr (PAIR) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w = 0;
      if (in0) w = __ldg(reinterpret_cast<const uint32_t*>(row + 2 * lane));  // R is even: both or none
      *reinterpret_cast<uint32_t*>(t.v) = w;
    } else {
      uint2 w = make_uint2(0, 0);
      if (in0) w = __ldg(reinterpret_cast<const uint2*>(row + 2 * lane));
      *reinterpret_cast<uint2*>(t.v) = w;
    }
  } else {
    t.v[0] = in0 ? row[lane] : St<T>::st(0.f);
    t.v[1] = in1 ? row[lane + 32] : St<T>::st(0.f);
  }
  return t;
}
// CTAs of an SM that the registers are held to: the loads of a CTA are all in flight at once, and other CTAs work meanwhile
// (8192 x 4096, bf16: 21.7 us with two, 18.3 with three, 19.7 with four; reading alone, in these 128-byte pieces, takes 17);
// the transcendental f need the registers.
__host__ __device__ constexpr int turned_ctas(size_t size, int act) {
  return size != 2 || (act != IPC_ACT_RELU && act != IPC_ACT_IDENTITY) ? 2 : 3;
}
template <typename T, int ACT, bool PAIR>
__global__ void __launch_bounds__(THREADS, turned_ctas(sizeof(T), ACT)) mx4_turned_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, int R, int K, int kp) {
  __shared__ __align__(16) unsigned char s_code[TUR][144];  // 128 bytes of codes per sample, rows 16 bytes apart mod 128
  __shared__ __align__(16) unsigned char s_scale[TUR][TB];
  const int r0 = blockIdx.x * TUR, k0 = blockIdx.y * TCOL;  // neighbouring CTAs read neighbouring samples
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kb = k0 + MX_BLOCK * warp;
  const int rl[2] = {PAIR ? 2 * lane : lane, PAIR ? 2 * lane + 1 : lane + 32};
  const bool in[2] = {r0 + rl[0] < R, r0 + rl[1] < R};
  const T* src = x + (long long)kb * R + r0;
  Two<T, PAIR> v[MX_BLOCK];
  if (kb + MX_BLOCK <= K) {
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i) v[i] = load_two<T, PAIR>(src + (long long)i * R, lane, in[0], in[1]);
  } else {
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i)
      v[i] = load_two<T, PAIR>(src + (long long)i * R, lane, in[0] && kb + i < K, in[1] && kb + i < K);
  }
  // 16-bit types under an f that only clears: both samples' largest magnitudes at once, as stored
  constexpr bool PACKED = sizeof(T) == 2 && (ACT == IPC_ACT_RELU || ACT == IPC_ACT_IDENTITY);
  uint32_t top[2] = {0, 0};
  if constexpr (PACKED) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i) {
      uint32_t& w = *reinterpret_cast<uint32_t*>(v[i].v);
      if constexpr (ACT == IPC_ACT_RELU) w = relu2<T>(w);
      m = __vmaxu2(m, w & 0x7fff7fffu);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t b = (uint16_t)(h ? m >> 16 : m & 0xffffu);
      top[h] = __float_as_uint(St<T>::ld(*reinterpret_cast<const T*>(&b)));
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[MX_BLOCK];
    if constexpr (!PACKED) {
#pragma unroll
      for (int i = 0; i < MX_BLOCK; ++i) {
        f[i] = mx_f<float, ACT>(St<T>::ld(v[i].v[h]));
        if (ACT == IPC_ACT_SIGMOID && !(in[h] && kb + i < K)) f[i] = 0.f;  // (the other f are 0 at 0)
        top[h] = max(top[h], f_bits<ACT>(f[i]));
      }
    }
    const uint32_t byte = mx4_scale_byte(top[h]);
    const float inv = mx_inv_scale(byte);
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float a[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = (PACKED ? St<T>::ld(v[8 * q + j].v[h]) : f[8 * q + j]) * inv;
      w[q] = byte == MX_NAN_BYTE ? 0u : mx4_pack8(a);
    }
    *reinterpret_cast<uint4*>(&s_code[rl[h]][16 * warp]) = o;
    s_scale[rl[h]][warp] = (unsigned char)byte;
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
__global__ void __launch_bounds__(threads_of(VEC)) mx4_restore_kernel(const unsigned char* __restrict__ codes,
                                                              const unsigned char* __restrict__ scales,
                                                              T* __restrict__ out, int R, int K, int kp) {
  const int r0 = blockIdx.y * TR, c0 = blockIdx.x * TCOL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if constexpr (VEC) {
    constexpr int N = 8, TPR = TCOL / N, RPI = THREADS / TPR, IT = TR / RPI;
    const int c = c0 + N * (tid % TPR), rf = r0 + tid / TPR;
    if (c >= K) return;
    // (a tile's 32 rows lie 16 bytes apart in their scale atom)
    const unsigned char* cp = codes + (long long)rf * (kp / 2) + c / 2;
    const unsigned char* sp = scales + mx4_scale_at(r0, c / MX_BLOCK, kp / 128) + 16 * (tid / TPR);
    T* op = out + (long long)rf * K + c;
    const long long cs = (long long)RPI * (kp / 2), os = (long long)RPI * K;
    uint32_t q[IT], byte[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {  // all loads first
      q[it] = byte[it] = 0;
      if (rf + RPI * it < R) {
        q[it] = __ldg(reinterpret_cast<const uint32_t*>(cp + it * cs));
        byte[it] = __ldg(sp + 16 * RPI * it);
      }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (rf + RPI * it >= R) break;
      const float sc = mx_scale(byte[it]);
      uint32_t h[4];
      mx4_unpack8(q[it], h);
      float v[N];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        v[2 * j] = f.x * sc;
        v[2 * j + 1] = f.y * sc;
      }
#pragma unroll
      for (int g = 0; g < N; g += Vec<T>::N)  // (K is a multiple of a vector)
        if (c + g < K) Vec<T>::store(op + it * os + g, *reinterpret_cast<float(*)[Vec<T>::N]>(v + g));
    }
  } else {
    constexpr int RW = TR / (LANE_THREADS / 32);
    uint32_t q[RW][TB], byte[RW][TB];
#pragma unroll
    for (int i = 0; i < RW; ++i)  // all loads first
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int r = r0 + warp + LANE_THREADS / 32 * i, c = c0 + MX_BLOCK * j + lane;
        const bool in = r < R && c < K;
        q[i][j] = in ? __ldg(codes + (long long)r * (kp / 2) + c / 2) : 0u;
        byte[i][j] = in ? __ldg(scales + mx4_scale_at(r, c / MX_BLOCK, kp / 128)) : 0u;
      }
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const int r = r0 + warp + LANE_THREADS / 32 * i, c = c0 + MX_BLOCK * j + lane;
        uint32_t h[4];
        mx4_unpack8((q[i][j] >> (4 * (lane & 1))) & 15u, h);
        if (r < R && c < K)
          out[(long long)r * K + c] =
              St<T>::st(__half2float(__ushort_as_half((unsigned short)(h[0] & 0xffffu))) * mx_scale(byte[i][j]));
      }
  }
}

// Rows of 16-bit elements copied to a stride that TMA takes: a thread stores 8 elements as one vector.
struct PackJob {
  const uint16_t* src;
  uint4* dst;
  int rows, n, ld8;
};
__device__ __forceinline__ void pack_rows(const PackJob& j, int block, int blocks) {
  const long long total = (long long)j.rows * j.ld8;
  for (long long i = block * (long long)THREADS + threadIdx.x; i < total; i += (long long)blocks * THREADS) {
    const int r = (int)(i / j.ld8), c = (int)(i % j.ld8) * 8;
    const uint16_t* p = j.src + (long long)r * j.n + c;
    uint4 v;
    uint16_t* h = reinterpret_cast<uint16_t*>(&v);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = c + k < j.n ? __ldg(p + k) : (uint16_t)0;
    j.dst[i] = v;
  }
}
int pack_blocks(const PackJob& j) {
  const long long n = ((long long)j.rows * j.ld8 + THREADS - 1) / THREADS;
  return (int)(n < 148 * 8 ? n : 148 * 8);
}
__global__ void __launch_bounds__(THREADS) mx8_pack_kernel(const PackJob a, const PackJob b, int blocks_a) {
  grid_let_next_start();
  if ((int)blockIdx.x < blocks_a)
    pack_rows(a, blockIdx.x, blocks_a);
  else
    pack_rows(b, blockIdx.x - blocks_a, gridDim.x - blocks_a);
}
// f(x^) of a checkpoint and the copy of another operand in one launch: the last `blocks_b` rows of blocks copy
template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS)
    mx8_restore_pack_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ scales,
                            T* __restrict__ out, int D, int cols, int nb, long long ld_out, const PackJob j, int rows_r, int* zero,
                            int n_zero) {
  grid_let_next_start();
  zero_words(zero, n_zero);
  if ((int)blockIdx.y < rows_r)
    restore_tile<T, ACT, true>(codes, scales, out, D, cols, nb, ld_out);
  else
    pack_rows(j, (blockIdx.y - rows_r) * gridDim.x + blockIdx.x, (gridDim.y - rows_r) * gridDim.x);
}

template <typename T>
bool rows_aligned(const void* p, long long ld) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (long long)sizeof(T))) & 15) == 0;
}

int lane_threads(const dim3& grid) { return (long long)grid.x * grid.y >= 296 ? THREADS : LANE_THREADS; }

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
      mx8_store_kernel<TT, false><<<grid, lane_threads(grid), 0, s>>>(xt, codes, scales, D, B, nb);
  });
  count_launch();
  return check_launch("8-bit store");
}

int launch_mx8_restore(const signed char* codes, const unsigned char* scales, void* out, int D, int B, long long ld_out,
                       int act, int dtype, cudaStream_t s, int* zero, int n_zero) {
  const int nb = (int)(mx8_ld(B) / MX_BLOCK);
  dim3 grid;
  int rc = grid_of("8-bit restore", D, TR, B, &grid);
  if (rc) return rc;
  IPC_DISPATCH_DT(dtype, TT, {
    TT* ot = static_cast<TT*>(out);
    const bool vec = rows_aligned<TT>(out, ld_out);
    IPC_DISPATCH_ACT(act, AC, {
      if (vec)
        mx8_restore_kernel<TT, AC, true><<<grid, THREADS, 0, s>>>(codes, scales, ot, D, B, nb, ld_out, zero, n_zero);
      else
        mx8_restore_kernel<TT, AC, false><<<grid, lane_threads(grid), 0, s>>>(codes, scales, ot, D, B, nb, ld_out, zero, n_zero);
    });
  });
  count_launch();
  return check_launch("8-bit restore");
}

int launch_mx8_pack(const void* src_a, void* dst_a, int rows_a, int n_a, long long ld_a, const void* src_b, void* dst_b,
                    int rows_b, int n_b, long long ld_b, cudaStream_t s) {
  const PackJob a{static_cast<const uint16_t*>(src_a), static_cast<uint4*>(dst_a), src_a ? rows_a : 0, n_a, (int)(ld_a / 8)};
  const PackJob b{static_cast<const uint16_t*>(src_b), static_cast<uint4*>(dst_b), src_b ? rows_b : 0, n_b, (int)(ld_b / 8)};
  const int blocks_a = src_a ? pack_blocks(a) : 0, blocks_b = src_b ? pack_blocks(b) : 0;
  if (blocks_a + blocks_b == 0) return IPC_OK;
  mx8_pack_kernel<<<blocks_a + blocks_b, THREADS, 0, s>>>(a, b, blocks_a);
  count_launch();
  return check_launch("row copy");
}

int launch_mx8_restore_pack(const signed char* codes, const unsigned char* scales, void* out, int D, int B,
                            long long ld_out, const void* src, void* dst, int rows, int act, int dtype, cudaStream_t s,
                            int* zero, int n_zero) {
  const int nb = (int)(mx8_ld(B) / MX_BLOCK);
  dim3 grid;
  const int rc = grid_of("8-bit restore", D, TR, B, &grid);
  if (rc) return rc;
  const PackJob j{static_cast<const uint16_t*>(src), static_cast<uint4*>(dst), rows, B, (int)(ld_out / 8)};
  const int rows_r = grid.y;
  long long extra = (pack_blocks(j) + grid.x - 1) / grid.x;
  if (rows_r + extra > 65535) extra = 65535 - rows_r;
  if (extra < 1) return set_error(IPC_ERR_ARG, "8-bit restore: %d rows are too many", D);
  grid.y += (unsigned)extra;
  IPC_DISPATCH_DT16(dtype, TT, {
    TT* ot = static_cast<TT*>(out);
    IPC_DISPATCH_ACT(act, AC, {
      mx8_restore_pack_kernel<TT, AC><<<grid, THREADS, 0, s>>>(codes, scales, ot, D, B, nb, ld_out, j, rows_r, zero,
                                                                 n_zero);
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
      if (turned && R % 2 == 0 && (reinterpret_cast<uintptr_t>(x) % (2 * sizeof(TT))) == 0)
        mx4_turned_kernel<TT, AC, true><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
      else if (turned)
        mx4_turned_kernel<TT, AC, false><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
      else if (vec)
        mx4_rows_kernel<TT, AC, true><<<grid, THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
      else
        mx4_rows_kernel<TT, AC, false><<<grid, LANE_THREADS, 0, s>>>(xt, codes, scales, R, K, kp);
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
      mx4_restore_kernel<TT, false><<<grid, LANE_THREADS, 0, s>>>(codes, scales, ot, R, K, kp);
  });
  count_launch();
  return check_launch("4-bit restore");
}

}  // namespace ipc
