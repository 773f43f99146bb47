// Microscaled storage: blocks of 32 numbers that share one power of two.
//
// A block whose largest magnitude is m is stored as a scale byte s + 127 and 32 codes c, each number
// standing for c * 2^s:
//   8 bits  s = the smallest integer with m <= 127 * 2^s; c = v * 2^-s rounded to the nearest integer
//   4 bits  s = the smallest integer with m <= 6 * 2^s;   c = v * 2^-s rounded to sign + {0, .5, 1, 1.5, 2, 3, 4, 6}
// (ties to even), s >= -127.  The scale is the smallest that clips nothing: the alternative for 4 bits that
// takes the exponent of m alone clips every m above 6 * 2^s by up to a quarter.  Scaling by a power of two is exact, so
// a code depends on the stored value alone, and c * 2^s is exact in bf16.  A block that holds an infinity or a
// NaN is stored as codes 0 with the scale byte 255 and reads back as 32 NaNs.
#pragma once
#include "ipc_common.cuh"
#include "ipc_generic.cuh"

namespace ipc {

constexpr int MX_BLOCK = 32;
constexpr uint32_t MX_NAN_BYTE = 255;

// Scale byte of a block from the bits of its largest magnitude (a non-negative float, or NaN).
// TOP_EXP / TOP_MANT: the exponent and mantissa field of the largest code (127 = 2^6 * 1.984375, 6 = 2^2 * 1.5).
template <int TOP_EXP, uint32_t TOP_MANT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return MX_NAN_BYTE;
  const int e = (int)(max_bits >> 23) - TOP_EXP + ((max_bits & 0x7fffffu) > TOP_MANT ? 1 : 0);
  return (uint32_t)max(e, 0);
}
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t max_bits) { return mx_scale_byte<6, 0x7e0000u>(max_bits); }
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t max_bits) { return mx_scale_byte<2, 0x400000u>(max_bits); }

// 2^s and 2^-s of a scale byte (2^-127 is a subnormal float; 255 stands for NaN and its codes for 0)
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == MX_NAN_BYTE ? 0x7fc00000u : byte << 23);
}
__device__ __forceinline__ float mx_inv_scale(uint32_t byte) {
  return byte == MX_NAN_BYTE ? 0.f : __uint_as_float((254u - byte) << 23);
}
// One 8-bit code.  A block marked NaN multiplies by 0: v * 0 is 0 or NaN, and NaN converts to 0.
__device__ __forceinline__ int mx8_code(float v, float inv) { return __float2int_rn(v * inv); }

// The four codes of a word as floats: a code + 128 in the low byte of 2^23's mantissa, less 2^23 + 128 (exact; two ALU
// operations each, where a conversion would take the slower pipe that f's MUFU forms need).
__device__ __forceinline__ void mx8_floats(uint32_t codes, float* v) {
  const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540u + i)) - 8388736.f;
}

// Eight numbers (already scaled, |v| <= 6) as 4-bit codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t mx4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint32_t mx4_pack2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tmov.b32 %0, {b, b, b, b};\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r & 0xffu;
}
// The inverse: eight 4-bit codes as four half2.
__device__ __forceinline__ void mx4_unpack8(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

// f and f' of states read back, in fp32, and f of what is quantised.  They are written with an exponential z of a negative
// number and r = 1 / (1 + z), so that no term is the small difference of large ones: f' of a saturated state and gelu of
// a negative one keep their relative accuracy (1 - tanh(x)^2 at x = 5, with tanh off by 2^-11, has no correct digit left;
// neither has 1 + tanh(u) in gelu at x = -4), and nothing overflows.
//   tanh'    = 4 z r^2            z = e^-2|x|
//   sigmoid' = z r^2              z = e^-|x|
//   silu'    = s + x z r^2        ... s = sigmoid(x) = r or z r
//   gelu     = x s                z = e^-2|u|, u = k (x + c x^3), s = sigmoid(2 u) = r or z r
//   gelu'    = s + 2 x u' z r^2
// In 16-bit storage z and r are ex2.approx and rcp.approx (2^-22 and 2^-23), in fp32 CUDA's expf and a division.  f' is off
// by about 2^-20 of itself, plus the exponent's rounding (its size times 2^-22).  tanh itself is tanh.approx in 16-bit
// storage, off by 2^-11 of itself, about one rounding of fp16.
// relu keeps a NaN: a block that held an infinity or a NaN reads back as NaNs, and taking those for 0 would hide it.
// T: the storage type.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGelu1 = 2.f * kGeluK, kGelu3 = 2.f * kGeluK * kGeluC;  // 2 u = x (kGelu1 + kGelu3 x^2)

__device__ __forceinline__ float mx_max_nan(float x, float y) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}
__device__ __forceinline__ float mx_min_nan(float x, float y) {
  float m;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}
__device__ __forceinline__ float mx_ex2(float x) {
  float z;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(z) : "f"(x));
  return z;
}
template <typename T>
__device__ __forceinline__ float mx_exp(float a, float x) {  // e^(a x), a x <= 0, a constant
  if constexpr (sizeof(T) == 2) return mx_ex2(a * kLog2e * x);
  return expf(a * x);
}
template <typename T>
__device__ __forceinline__ float mx_recip(float x) {  // 1 <= x <= 2 in fp32
  if constexpr (sizeof(T) == 2) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
  }
  return __fdividef(1.f, x);
}

template <typename T, int ACT>
__device__ __forceinline__ float mx_f(float x) {
  if constexpr (ACT == IPC_ACT_RELU) {
    return mx_max_nan(x, 0.f);  // (one instruction, where a comparison that lets NaN through takes two)
  } else if constexpr (ACT == IPC_ACT_GELU) {
    if constexpr (sizeof(T) == 2) {
      return x * mx_recip<T>(1.f + mx_ex2(x * fmaf(-kGelu3 * kLog2e, x * x, -kGelu1 * kLog2e)));  // (z of either sign)
    }
    const float z = mx_exp<T>(-1.f, fabsf(x) * fmaf(kGelu3, x * x, kGelu1));
    return x * (x >= 0.f ? 1.f : z) * mx_recip<T>(1.f + z);
  } else if constexpr (sizeof(T) == 2) {
    return act_f_hw<ACT>(x);
  } else if constexpr (ACT == IPC_ACT_SIGMOID || ACT == IPC_ACT_SILU) {
    // 1 / (1 + e^-x) itself is 0 below x = -88.7, where sigmoid(x) is still a (subnormal) number.  Far below 0 silu is x e^x,
    // whose e^x alone would be rounded as a subnormal before x multiplies it: the last factor e^-32 comes at the end.
    if (ACT == IPC_ACT_SILU && x < -64.f) return x * expf(x + 32.f) * 1.26641655e-14f;
    const float z = expf(-fabsf(x));
    const float n = x >= 0.f ? 1.f : z;
    return (ACT == IPC_ACT_SILU ? x * n : n) / (1.f + z);
  } else {
    return act_f<ACT>(x);
  }
}
template <typename T, int ACT>
__device__ __forceinline__ float mx_df(float x) {
  if constexpr (ACT == IPC_ACT_TANH) {
    const float z = mx_exp<T>(-2.f, fabsf(x)), r = mx_recip<T>(1.f + z);
    return 4.f * z * r * r;
  } else if constexpr (ACT == IPC_ACT_SIGMOID || ACT == IPC_ACT_SILU || ACT == IPC_ACT_GELU) {
    // (from |x| = 20 on z is 0, and 0 times the infinite square of a large x would be no number)
    const float x2 = ACT == IPC_ACT_GELU ? fminf(x * x, 400.f) : 0.f;
    const float z = ACT == IPC_ACT_GELU ? mx_exp<T>(-1.f, fabsf(x) * fmaf(kGelu3, x2, kGelu1)) : mx_exp<T>(-1.f, fabsf(x));
    const float r = mx_recip<T>(1.f + z), zr = z * r, d = zr * r;
    if constexpr (ACT == IPC_ACT_SIGMOID) return d;
    const float s = x >= 0.f ? r : zr;
    return fmaf(ACT == IPC_ACT_SILU ? x : x * fmaf(3.f * kGelu3, x2, kGelu1), d, s);
  } else {
    return act_df<ACT>(x);
  }
}

// f'(c * 2^s) for the codes of a block: what depends on its step 2^s alone is the same for all of them (relu's NaN; the exponents of
// tanh' and sigmoid', which take |c|, and tanh's 4 as the exponent's 2).
template <typename T, int ACT>
__device__ __forceinline__ float mx_df_code(float c, float step) {
  if constexpr (ACT == IPC_ACT_RELU) {
    return (c > 0.f ? 1.f : 0.f) + step * 0.f;
  } else if constexpr (sizeof(T) == 2 && (ACT == IPC_ACT_TANH || ACT == IPC_ACT_SIGMOID)) {
    const float a = mx_max_nan((ACT == IPC_ACT_TANH ? -2.f : -1.f) * kLog2e * step, -3e38f);  // (0 times infinity is no number)
    if constexpr (ACT == IPC_ACT_TANH) {
      const float z4 = mx_ex2(fmaf(fabsf(c), a, 2.f)), r = mx_recip<T>(fmaf(0.25f, z4, 1.f));
      return z4 * r * r;
    }
    const float z = mx_ex2(fabsf(c) * a), r = mx_recip<T>(1.f + z);
    return z * r * r;
  } else {
    return mx_df<T, ACT>(c * step);
  }
}

// Layouts.  8 bits: codes [D][32 * ceil(B/32)], scale bytes [ceil(B/32)][D], blocks along the batch.
// 4 bits, R rows of K columns: codes [R][Kp/2], Kp = 128 * ceil(K/128), lower column in the lower nibble; scale
// bytes in atoms of 128 rows x 4 blocks, [ceil(R/128)][Kp/128][32][4][4] with row r, block j at
// [r/128][j/4][r%32][r%128/32][j%4] (what the tensor core's scale operand takes).
__host__ __device__ inline long long mx8_ld(int B) { return ((long long)B + 31) / 32 * 32; }
__host__ __device__ inline long long mx4_kp(int K) { return ((long long)K + 127) / 128 * 128; }
__device__ __forceinline__ long long mx4_scale_at(int r, int j, int atoms_k) {
  return ((long long)(r >> 7) * atoms_k + (j >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (j & 3);
}

// The largest of 16, 8, 4 and 2 bytes that divides an address and a row stride.
inline int row_alignment(const void* p, long long row_bytes) {
  const unsigned long long bits = reinterpret_cast<unsigned long long>(p) | (unsigned long long)row_bytes;
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

int launch_mx8_store(const void* x, signed char* codes, unsigned char* scales, int D, int B, int dtype, cudaStream_t s);
// out[d][b] = cast(f(codes * 2^s)), rows ld_out >= B apart; n_zero words at `zero` are cleared beside it
int launch_mx8_restore(const signed char* codes, const unsigned char* scales, void* out, int D, int B, long long ld_out,
                       int act, int dtype, cudaStream_t s, int* zero = nullptr, int n_zero = 0);
// Up to two copies dst [rows][ld] = src [rows][n] of 16-bit elements in one launch (a null src: none; ld a multiple of 8,
// dst 16-byte aligned, columns n .. ld - 1 zeroed)
int launch_mx8_pack(const void* src_a, void* dst_a, int rows_a, int n_a, long long ld_a, const void* src_b, void* dst_b,
                    int rows_b, int n_b, long long ld_b, cudaStream_t s);
// launch_mx8_restore and such a copy of src [rows][B] to the same stride, in one launch (16-bit storage)
int launch_mx8_restore_pack(const signed char* codes, const unsigned char* scales, void* out, int D, int B,
                            long long ld_out, const void* src, void* dst, int rows, int act, int dtype, cudaStream_t s,
                            int* zero = nullptr, int n_zero = 0);
// one-launch product with a checkpoint (p.ck, p.cks), any shape, 16-bit storage: MODE_W, _WD, _G, _BK
int launch_mx8_small(const GemmArgs& p, int mode, int act, int dtype, cudaStream_t s);
// the same for a few samples (1 to 16; MODE_BK 1 to 4), any storage type, in fp32
int launch_mx8_few(const GemmArgs& p, int mode, int act, int dtype, cudaStream_t s);
int launch_mx4_quantize(const void* x, unsigned char* codes, unsigned char* scales, int R, int K, int turned, int act,
                        int dtype, cudaStream_t s);
int launch_mx4_restore(const unsigned char* codes, const unsigned char* scales, void* out, int R, int K, int dtype,
                       cudaStream_t s);
int launch_mx4_gemm(const unsigned char* w, const unsigned char* ws, const unsigned char* a, const unsigned char* as,
                    void* out, int M, int K, int B, int dtype, cudaStream_t s);
// First error a bounded wait of the 4-bit product recorded (0 = none); clear != 0 resets it.
int read_mx_status(int* status, int clear);

}  // namespace ipc
