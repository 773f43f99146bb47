// out [M, B] = W4 [M, K] @ A4 [B, K]^T for 4-bit operands in blocks of 32 along K (ipc_mx.cuh).
//
// The tensor core multiplies the 4-bit codes as they are stored and applies both scale bytes itself
// (tcgen05.mma.kind::mxf4.block_scale): the products are exact and the sums fp32.
//
// One persistent CTA per SM (or as many as ipc_set_max_ctas leaves) walks output tiles of 128 x BN.  (CTA pairs, 256 x 256 tiles, were slower: 76 us against 69
// at 4096 x 4096 x 8192 with tcgen05.cp, and 127 against 60 with the scale warps, whose signal then crosses SMs.)
// Warp 0 loads K blocks of 256 columns (128 bytes a row, 128-byte swizzle) and their scale atoms with TMA into a
// ring of stages; warps 10..13 put a stage's scale factors into tensor memory, each into its lane quarter; warp 1 issues the
// stage's four MMAs; warps 2..9 read the accumulator, and write it through a swizzled buffer in shared memory, so that
// a warp stores whole 64-byte row pieces.
//
// Scale factors: the MMA takes those of 128 rows x 4 blocks from 4 columns, in each lane quarter lane i, column c the
// bytes of row 32 c + i: 16 bytes of an atom a lane, so a warp moves an atom with one 16-byte load and one tcgen05.st.
// tcgen05.cp would do it in one instruction of the MMA thread, but runs in order with the MMAs: six copies before a
// stage's four MMAs made 4096 x 4096 x 8192 take 69 us instead of 60 (74 to 77 with the copies a stage ahead).
//
// Tensor memory: 512 columns hold the scale factors of two stages (24 columns each at most) and two accumulators, so
// that a tile's epilogue runs beside the next tile's MMAs.  Two of 256 columns leave no room: they overlap in 64
// columns (0 .. 255 and 192 .. 447), which the epilogue reads first; the next tile starts once they are read.
#include <cudaTypedefs.h>

#include <cstring>
#include <mutex>
#include <type_traits>

#include "ipc_mx.cuh"
#include "ipc_ptx.cuh"
#include "ipc_tc.cuh"

namespace ipc {

__device__ int g_mx_status = 0;  // first error code a bounded wait of this file raised

namespace {

constexpr int F_BM = 128;                // rows of a CTA's tile
constexpr int F_BK = 256;                // columns of a stage
constexpr int F_KB = F_BK / 2;           // ... in bytes: one 128-byte swizzle row
constexpr int F_EPI_WARPS = 8;           // two per TMEM lane quarter, one per half of the accumulator's columns
constexpr int F_SF_WARPS = 4;
constexpr int F_THREADS = 64 + 32 * (F_EPI_WARPS + F_SF_WARPS);
constexpr int F_EPI_BYTES = 2048;        // per warp: 32 rows x 64 bytes
constexpr int F_SF_BUFS = 2;             // scale factors of two stages in tensor memory
constexpr uint32_t F_SF_COLS = 32;       // columns of one buffer (24 used)
constexpr uint32_t F_SF_COL = 448;       // the first
constexpr uint32_t F_ATOM = 512;         // bytes of a scale atom: 128 rows x 4 blocks

__host__ __device__ constexpr int f_stage_bytes(int bn) { return (F_BM + bn) * F_KB + (1 + bn / 128) * 2 * (int)F_ATOM; }
__host__ __device__ constexpr int f_stages(int bn) { return bn == 256 ? 4 : 5; }
__host__ __device__ constexpr int f_acc_col(int bn) { return bn == 256 ? 192 : bn; }  // second accumulator

struct Mx4Params {
  int M, N, nk;  // nk: stages of 256 columns
  int tiles_m, tiles_n, tiles, raster;
  void* out;
  long long ld_out;
  int vec;  // bytes of a store: the largest of 16, 8, 4, 2 on whose boundaries the rows of out start
};

__device__ __forceinline__ bool f_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait_bounded(bar, parity, abort_flag, &g_mx_status);
}
__device__ __forceinline__ void f_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// the 16 bytes a lane holds of each of N / 4 scale atoms -> N columns of the warp's lane quarter
template <int N>
__device__ __forceinline__ void f_store_scales(uint32_t tmem, const uint32_t (&r)[N]) {
  static_assert(N == 8 || N == 16, "");
  if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(tmem), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  else
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(tmem),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// two chunks of 32 accumulator columns, one wait
__device__ __forceinline__ void f_read64(uint32_t taddr, uint32_t (&r)[64]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[32 * h]), "=r"(r[32 * h + 1]), "=r"(r[32 * h + 2]), "=r"(r[32 * h + 3]), "=r"(r[32 * h + 4]),
          "=r"(r[32 * h + 5]), "=r"(r[32 * h + 6]), "=r"(r[32 * h + 7]), "=r"(r[32 * h + 8]), "=r"(r[32 * h + 9]),
          "=r"(r[32 * h + 10]), "=r"(r[32 * h + 11]), "=r"(r[32 * h + 12]), "=r"(r[32 * h + 13]), "=r"(r[32 * h + 14]),
          "=r"(r[32 * h + 15]), "=r"(r[32 * h + 16]), "=r"(r[32 * h + 17]), "=r"(r[32 * h + 18]), "=r"(r[32 * h + 19]),
          "=r"(r[32 * h + 20]), "=r"(r[32 * h + 21]), "=r"(r[32 * h + 22]), "=r"(r[32 * h + 23]), "=r"(r[32 * h + 24]),
          "=r"(r[32 * h + 25]), "=r"(r[32 * h + 26]), "=r"(r[32 * h + 27]), "=r"(r[32 * h + 28]), "=r"(r[32 * h + 29]),
          "=r"(r[32 * h + 30]), "=r"(r[32 * h + 31])
        : "r"(taddr + 32 * h));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void f_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                      uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc));
}

// Tile t -> first row of the unit's tile and first column; rows in bands of `raster` tiles, all columns of a band first.
__device__ __forceinline__ void f_tile(const Mx4Params& p, int t, int bn, int& m0, int& n0) {
  const int band = t / (p.raster * p.tiles_n);
  const int first = band * p.raster;
  const int rows = min(p.raster, p.tiles_m - first);
  const int within = t - band * p.raster * p.tiles_n;
  m0 = (first + within % rows) * F_BM;
  n0 = (within / rows) * bn;
}

template <typename T, int BN>
__global__ void __launch_bounds__(F_THREADS, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                    const __grid_constant__ Mx4Params p) {
  constexpr int STAGES = f_stages(BN);
  constexpr uint32_t A_BYTES = F_BM * F_KB, B_BYTES = BN * F_KB;
  constexpr uint32_t STAGE_BYTES = f_stage_bytes(BN);
  constexpr int RB = BN / 128;  // row blocks of B's scale atoms
  constexpr uint32_t ACC1 = f_acc_col(BN);
  constexpr bool OVERLAP = BN == 256;
  // instruction descriptor: both operands 4-bit (e2m1), K-major, power-of-two scales; bits 4-5 / 29-30 choose the
  // two of an atom's four blocks that an MMA's 64 columns take
  constexpr uint32_t IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (1u << 23) | ((uint32_t)(F_BM >> 4) << 24);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + F_EPI_WARPS * F_EPI_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 6 + F_SF_BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full0 = saddr(bars), empty0 = saddr(bars + STAGES);
  // accumulator ready, accumulator read, overlapped columns read; scale factors in tensor memory
  const uint32_t tfull0 = saddr(bars + 2 * STAGES), tempty0 = tfull0 + 16, tover0 = tfull0 + 32, sready0 = tfull0 + 48;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tempty0 + 8 * b, F_EPI_WARPS);
      mbar_init(tover0 + 8 * b, F_EPI_WARPS / 2);
    }
    for (int b = 0; b < F_SF_BUFS; ++b) mbar_init(sready0 + 8 * b, F_SF_WARPS);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        int m0, n0;
        f_tile(p, t, BN, m0, n0);
        for (int kb = 0; kb < p.nk; ++kb) {
          ok = f_wait(empty0 + 8 * s, phase ^ 1, abort_flag);
          if (!ok) break;
          const uint32_t sa = saddr(smem + s * STAGE_BYTES), sb = sa + A_BYTES, ssa = sb + B_BYTES, ssb = ssa + 2 * F_ATOM;
          const uint32_t bar = full0 + 8 * s;
          mbar_expect_tx(bar, STAGE_BYTES);
          f_load(ssa, &tmSA, bar, kb * 256, m0 / 128);
          f_load(ssb, &tmSB, bar, kb * 256, n0 / 128);
          f_load(sa, &tmA, bar, kb * F_KB, m0);
          f_load(sb, &tmB, bar, kb * F_KB, n0);
          if (++s == STAGES) { s = 0; phase ^= 1; }
          ++issued;
        }
      }
      if (!ok) {  // loads in flight land (or 1 ms passes) before the CTA gives up its shared memory
        for (int k = 0; k < STAGES && k < issued; ++k) {
          const int it = issued - 1 - k;
          mbar_drain(full0 + 8 * (it % STAGES), (it / STAGES) & 1);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer -------------------------------
    if (lane == 0) {
      int s = 0, i = 0, it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x, ++i) {
        const int b = i & 1;
        ok = f_wait(tempty0 + 8 * b, ((i >> 1) & 1) ^ 1, abort_flag);
        if (OVERLAP && ok && i > 0) ok = f_wait(tover0 + 8 * (b ^ 1), ((i - 1) >> 1) & 1, abort_flag);
        if (!ok) break;
        const uint32_t d = tmem + b * ACC1;
        for (int kb = 0; kb < p.nk; ++kb, ++it) {
          // the scale warps signal after they have seen the stage's loads land
          ok = f_wait(sready0 + 8 * (it % F_SF_BUFS), (it / F_SF_BUFS) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = saddr(smem + s * STAGE_BYTES), sb = sa + A_BYTES;
          const uint32_t csa = tmem + F_SF_COL + F_SF_COLS * (it % F_SF_BUFS), csb = csa + 8;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t id = (kk & 1) * 2;
            f_mma(d, smem_desc(sa + kk * 32, 16, 1024), smem_desc(sb + kk * 32, 16, 1024), IDESC | (id << 4) | (id << 29),
                  csa + 4 * (kk >> 1), csb + 4 * RB * (kk >> 1), (kb > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(empty0 + 8 * s);
          if (++s == STAGES) s = 0;
        }
        if (!ok) break;
        tc_commit(tfull0 + 8 * b);
      }
    }
    __syncwarp();
  } else if (warp >= 2 + F_EPI_WARPS) {
    // -------------------- scale factors: shared -> tensor memory --------------------
    const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16;
    int s = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
      for (int kb = 0; kb < p.nk; ++kb, ++it) {
        ok = f_wait(full0 + 8 * s, phase, abort_flag);
        const int prev = it - F_SF_BUFS;  // the MMAs that read this buffer are done once their stage is released
        if (ok && prev >= 0) ok = f_wait(empty0 + 8 * (prev % STAGES), (prev / STAGES) & 1, abort_flag);
        __syncwarp();
        if (!ok) break;
        const uint32_t ssa = saddr(smem + s * STAGE_BYTES) + A_BYTES + B_BYTES + 16 * lane, ssb = ssa + 2 * F_ATOM;
        uint32_t ra[8], rb[8 * RB];
#pragma unroll
        for (int ka = 0; ka < 2; ++ka) {
          const uint4 v = lds128(ssa + ka * F_ATOM);
          ra[4 * ka] = v.x; ra[4 * ka + 1] = v.y; ra[4 * ka + 2] = v.z; ra[4 * ka + 3] = v.w;
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            const uint4 u = lds128(ssb + (2 * r + ka) * F_ATOM);
            const int o = 4 * RB * ka + 4 * r;
            rb[o] = u.x; rb[o + 1] = u.y; rb[o + 2] = u.z; rb[o + 3] = u.w;
          }
        }
        const uint32_t col = tmem + quarter + F_SF_COL + F_SF_COLS * (it % F_SF_BUFS);
        tc_fence_after();
        f_store_scales<8>(col, ra);
        f_store_scales<8 * RB>(col + 8, rb);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sready0 + 8 * (it % F_SF_BUFS));
        if (++s == STAGES) { s = 0; phase ^= 1; }
      }
    }
  } else {
    // ------------------------------- epilogue --------------------------------
    const int q = warp & 3, half = (warp - 2) >> 2;
    constexpr int HC = BN / 2, NPASS = HC / 64;
    constexpr int EW = sizeof(T) == 4 ? 16 : 32;  // columns of one pass through the buffer: 64 bytes a row
    const uint32_t xb = saddr(smem + STAGES * STAGE_BYTES) + (warp - 2) * F_EPI_BYTES;
    T* out = reinterpret_cast<T*>(p.out);
    int i = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
      int m0, n0;
      f_tile(p, t, BN, m0, n0);
      const int r0 = m0 + 32 * q;
      const int b = i & 1;
      const bool ok = f_wait(tfull0 + 8 * b, (i >> 1) & 1, abort_flag);
      __syncwarp();
      if (!ok) break;
      tc_fence_after();
      const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + b * ACC1 + half * HC;
      const bool over = OVERLAP && half != b;  // this warp's half holds the overlapped columns: its last or first 64
#pragma unroll 1
      for (int ps = 0; ps < NPASS; ++ps) {
        const int c = (over && b == 0) ? NPASS - 1 - ps : ps;
        uint32_t raw[64];
        f_read64(trow + 64 * c, raw);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (over && ps == 0) mbar_arrive(tover0 + 8 * b);
          if (ps == NPASS - 1) mbar_arrive(tempty0 + 8 * b);
        }
        const int n = n0 + half * HC + 64 * c;
        if (r0 >= p.M || n >= p.N) continue;
#pragma unroll
        for (int e = 0; e < 64 / EW; ++e) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // row = lane: four vectors of 16 bytes, vector index ^ (row >> 1)
            uint4 v;
            if constexpr (sizeof(T) == 4) {
              v = make_uint4(raw[16 * e + 4 * j], raw[16 * e + 4 * j + 1], raw[16 * e + 4 * j + 2], raw[16 * e + 4 * j + 3]);
            } else {
              T* h = reinterpret_cast<T*>(&v);
#pragma unroll
              for (int k = 0; k < 8; ++k) h[k] = St<T>::st(__uint_as_float(raw[32 * e + 8 * j + k]));
            }
            sts128(xb + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), v);
          }
          __syncwarp();
          const int ne = n + EW * e;
          char* dst = reinterpret_cast<char*>(out + (long long)r0 * p.ld_out + ne);
          const long long ld = p.ld_out * (long long)sizeof(T);
          const int rows = p.M - r0, bytes = min(p.N - ne, EW) * (int)sizeof(T);
          auto swz = [](int r) { return (r >> 1) & 3; };
          switch (p.vec) {
            case 16: store_rows<64, 16>(dst, ld, rows, bytes, xb, lane, swz); break;
            case 8: store_rows<64, 8>(dst, ld, rows, bytes, xb, lane, swz); break;
            case 4: store_rows<64, 4>(dst, ld, rows, bytes, xb, lane, swz); break;
            default:
              if constexpr (sizeof(T) == 2) store_rows<64, 2>(dst, ld, rows, bytes, xb, lane, swz);
          }
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ----------------------------------------------------------------------------------- few samples
// A whole tile of the kernel above costs its set-up (8 us for a single sample) whatever it holds.  Here a warp owns 16
// rows x 8 NB samples and a part of K; codes go from global memory to registers, are widened to fp16 (exact) and multiplied by
// mma.sync a block of 32 columns at a time (two MMAs into zeros), and the block's sum c (up to 1152) is scaled into the fp32
// accumulator: (c * 2^sw) * 2^sa.  Where 2^sw is so large that this could overflow though 2^sa brings it back, the smaller
// scale comes first (c * 2^-127 is still exact, c a multiple of 1/4; always doing so takes 4096 x 4096 x 1 from 7.4 us
// to 7.9).  Which of a block's columns an MMA's k stands for is free as long
// as both operands agree, so lane t of a quad takes 8 neighbouring columns: 4 bytes of each row.  The KW warps of a row block add up in
// shared memory in warp order.  One read of W: 4096 x 4096 x 1 is 8.9 MB.
constexpr int G_WARPS = 8;

__device__ __forceinline__ void g_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// acc + c * 2^s0 * 2^s1; with LARGE the smaller scale first (positive floats compare as their bits do, NaN above all)
template <bool LARGE>
__device__ __forceinline__ float g_scaled(float acc, float c, float s0, float s1) {
  const uint32_t a = __float_as_uint(s0), b = __float_as_uint(s1);
  if constexpr (LARGE) return fmaf(c * __uint_as_float(min(a, b)), __uint_as_float(max(a, b)), acc);
  return fmaf(c * s0, s1, acc);
}
// whether one of four scale bytes is 240 (2^113) or more
__device__ __forceinline__ bool g_large(uint32_t bytes) {
  const uint32_t two = bytes & (bytes >> 1);
  return (two & (two >> 2) & 0x10101010u) != 0;
}
// the four scale bytes of an atom's row (0 for a row past the operand: its codes are not read either)
__device__ __forceinline__ uint32_t g_scales(const unsigned char* sc, int r, int rows, int atom, int atoms) {
  return r < rows ? __ldg(reinterpret_cast<const uint32_t*>(sc + mx4_scale_at(r, 4 * atom, atoms))) : 0u;
}

template <typename T, int NB>
__global__ void __launch_bounds__(32 * G_WARPS)
    mx4_small_kernel(const unsigned char* __restrict__ w, const unsigned char* __restrict__ wsc,
                     const unsigned char* __restrict__ a, const unsigned char* __restrict__ asc, T* __restrict__ out,
                     int M, int B, int kp, int kw) {
  __shared__ float red[G_WARPS][16][8 * NB + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = warp % kw;  // this warp's share of K
  const int m0 = (blockIdx.x * (G_WARPS / kw) + warp / kw) * 16, n0 = blockIdx.y * 8 * NB;
  const int atoms = kp / 128, ldc = kp / 2;
  float acc[NB][4] = {};
  const unsigned char* w0 = w + (long long)(m0 + g) * ldc + 4 * t;
  const unsigned char* w1 = w0 + 8LL * ldc;
  const bool in0 = m0 + g < M, in1 = m0 + g + 8 < M;
  struct Atom {
    uint32_t cw[4][2], ca[4][NB], sw[2], sa[NB][2];
  };
  auto fetch = [&](Atom& f, int at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = 64 * at + 16 * j;
      f.cw[j][0] = in0 ? __ldg(reinterpret_cast<const uint32_t*>(w0 + o)) : 0u;
      f.cw[j][1] = in1 ? __ldg(reinterpret_cast<const uint32_t*>(w1 + o)) : 0u;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int n = n0 + 8 * b + g;
        f.ca[j][b] = n < B ? __ldg(reinterpret_cast<const uint32_t*>(a + (long long)n * ldc + 4 * t + o)) : 0u;
      }
    }
    f.sw[0] = g_scales(wsc, m0 + g, M, at, atoms);
    f.sw[1] = g_scales(wsc, m0 + g + 8, M, at, atoms);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f.sa[b][0] = g_scales(asc, n0 + 8 * b + 2 * t, B, at, atoms);
      f.sa[b][1] = g_scales(asc, n0 + 8 * b + 2 * t + 1, B, at, atoms);
    }
  };
  Atom cur, next;
  if (part < atoms) fetch(cur, part);
  for (int at = part; at < atoms; at += kw) {
    if (at + kw < atoms) fetch(next, at + kw);  // the next atom's loads under this one's MMAs
    auto atom = [&](auto large) {
      constexpr bool LARGE = decltype(large)::value;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t x0[4], x1[4];
        mx4_unpack8(cur.cw[j][0], x0);
        mx4_unpack8(cur.cw[j][1], x1);
        const float f0 = mx_scale((cur.sw[0] >> (8 * j)) & 255u), f1 = mx_scale((cur.sw[1] >> (8 * j)) & 255u);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t y[4];
          mx4_unpack8(cur.ca[j][b], y);
          float c[4] = {};
          g_mma(c, x0[0], x1[0], x0[1], x1[1], y[0], y[1]);
          g_mma(c, x0[2], x1[2], x0[3], x1[3], y[2], y[3]);
          const float h0 = mx_scale((cur.sa[b][0] >> (8 * j)) & 255u), h1 = mx_scale((cur.sa[b][1] >> (8 * j)) & 255u);
          acc[b][0] = g_scaled<LARGE>(acc[b][0], c[0], f0, h0);
          acc[b][1] = g_scaled<LARGE>(acc[b][1], c[1], f0, h1);
          acc[b][2] = g_scaled<LARGE>(acc[b][2], c[2], f1, h0);
          acc[b][3] = g_scaled<LARGE>(acc[b][3], c[3], f1, h1);
        }
      }
    };
    // (the same for all lanes: an MMA is the whole warp's)
    if (__any_sync(0xffffffffu, g_large(cur.sw[0]) || g_large(cur.sw[1]))) atom(std::true_type{});
    else atom(std::false_type{});
    cur = next;
  }
  if (kw > 1) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[warp][g + (r >= 2 ? 8 : 0)][8 * b + 2 * t + (r & 1)] = acc[b][r];
    __syncthreads();
    for (int i = threadIdx.x; i < G_WARPS / kw * 16 * 8 * NB; i += 32 * G_WARPS) {
      const int n = i % (8 * NB), r = i / (8 * NB) % 16, rb = i / (16 * 8 * NB);
      const int m = (blockIdx.x * (G_WARPS / kw) + rb) * 16 + r;
      float sum = 0.f;
      for (int k = 0; k < kw; ++k) sum += red[rb * kw + k][r][n];
      if (m < M && n0 + n < B) out[(long long)m * B + n0 + n] = St<T>::st(sum);
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + g + (r >= 2 ? 8 : 0), n = n0 + 8 * b + 2 * t + (r & 1);
        if (m < M && n < B) out[(long long)m * B + n] = St<T>::st(acc[b][r]);
      }
  }
}

template <typename T>
int launch_few(const unsigned char* w, const unsigned char* wsc, const unsigned char* a, const unsigned char* asc,
               void* out, int M, int K, int B, cudaStream_t s) {
  const int kp = (int)mx4_kp(K), atoms = kp / 128;
  const int kw = atoms >= 8 ? 8 : atoms >= 4 ? 4 : atoms >= 2 ? 2 : 1;
  const int rows = 16 * (G_WARPS / kw);
  const int nb = B <= 8 ? 1 : 2;
  const dim3 grid((unsigned)((M + rows - 1) / rows), (unsigned)((B + 8 * nb - 1) / (8 * nb)));
  T* o = static_cast<T*>(out);
  if (nb == 1)
    mx4_small_kernel<T, 1><<<grid, 32 * G_WARPS, 0, s>>>(w, wsc, a, asc, o, M, B, kp, kw);
  else
    mx4_small_kernel<T, 2><<<grid, 32 * G_WARPS, 0, s>>>(w, wsc, a, asc, o, M, B, kp, kw);
  count_launch();
  return check_launch("4-bit product of few samples");
}

// ------------------------------------------------------------------------------------------ host
PFN_cuTensorMapEncodeTiled_v12000 f_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// codes [rows][bytes]: boxes of box_rows x 128 bytes, 128-byte swizzle
int f_map_codes(CUtensorMap* map, const void* base, long long bytes, long long rows, int box_rows) {
  auto fn = f_encode();
  if (fn == nullptr) return set_error(IPC_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)bytes};
  const cuuint32_t box[2] = {(cuuint32_t)F_KB, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? IPC_OK : set_error(IPC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}
// scale atoms [row blocks][atoms * 512 bytes] as 32-bit words: boxes of box_rows row blocks x two atoms
int f_map_scales(CUtensorMap* map, const void* base, long long atoms, long long blocks, int box_rows) {
  auto fn = f_encode();
  if (fn == nullptr) return set_error(IPC_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)(atoms * 128), (cuuint64_t)blocks};
  const cuuint64_t strides[1] = {(cuuint64_t)(atoms * 512)};
  const cuuint32_t box[2] = {256, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? IPC_OK : set_error(IPC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

template <typename T, int BN>
int launch_tiles(const unsigned char* w, const unsigned char* wsc, const unsigned char* a, const unsigned char* asc,
                 void* out, int M, int K, int B, cudaStream_t s) {
  const long long kp = mx4_kp(K);
  CUtensorMap ta, tb, tsa, tsb;
  int rc = f_map_codes(&ta, w, kp / 2, M, F_BM);
  if (!rc) rc = f_map_codes(&tb, a, kp / 2, B, BN);
  if (!rc) rc = f_map_scales(&tsa, wsc, kp / 128, (M + 127) / 128, 1);
  if (!rc) rc = f_map_scales(&tsb, asc, kp / 128, (B + 127) / 128, BN / 128);
  if (rc) return rc;
  Mx4Params p{};
  p.M = M;
  p.N = B;
  p.nk = (int)((kp + F_BK - 1) / F_BK);
  p.tiles_m = (M + F_BM - 1) / F_BM;
  p.tiles_n = (B + BN - 1) / BN;
  p.tiles = p.tiles_m * p.tiles_n;
  p.raster = 16;
  p.out = out;
  p.ld_out = B;
  p.vec = row_alignment(out, (long long)B * (long long)sizeof(T));
  constexpr int SMEM = f_stages(BN) * f_stage_bytes(BN) + F_EPI_WARPS * F_EPI_BYTES + 1024 + 256;
  static_assert(SMEM <= 232448, "shared memory of a 4-bit product CTA");
  cudaError_t err = ensure_kernel_smem<mx4_gemm_kernel<T, BN>>(SMEM);
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "4-bit product smem attribute: %s", cudaGetErrorString(err));
  const int sms = grid_cap();
  mx4_gemm_kernel<T, BN><<<p.tiles < sms ? p.tiles : sms, F_THREADS, SMEM, s>>>(ta, tb, tsa, tsb, p);
  count_launch();
  return check_launch("4-bit product");
}

template <typename T>
__global__ void zero_kernel(T* out, long long n) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
    out[i] = St<T>::st(0.f);
}

}  // namespace

int launch_mx4_gemm(const unsigned char* w, const unsigned char* wsc, const unsigned char* a, const unsigned char* asc,
                    void* out, int M, int K, int B, int dtype, cudaStream_t s) {
  // Tile width: every CTA takes ceil(tiles / SMs) tiles; a 128-column tile takes 0.75 of a 256-column tile's time
  // (4096 x 4096 x 8192: 14 rounds in 90 us against 7 in 60), so 256 columns unless 128 save a quarter of the rounds.
  const long long sms = grid_cap(), tm = (M + 127) / 128;
  const long long w256 = (tm * ((B + 255) / 256) + sms - 1) / sms, w128 = (tm * ((B + 127) / 128) + sms - 1) / sms;
  const bool wide = B > 128 && 4 * w256 <= 3 * w128;
  IPC_DISPATCH_DT(dtype, TT, {
    if (K == 0) {
      zero_kernel<TT><<<148, 256, 0, s>>>(static_cast<TT*>(out), (long long)M * B);
      count_launch();
      return check_launch("4-bit product of no columns");
    }
    if (B <= 16) return launch_few<TT>(w, wsc, a, asc, out, M, K, B, s);
    return wide ? launch_tiles<TT, 256>(w, wsc, a, asc, out, M, K, B, s)
                : launch_tiles<TT, 128>(w, wsc, a, asc, out, M, K, B, s);
  });
  return IPC_OK;
}

int read_mx_status(int* status, int clear) {
  int v = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&v, g_mx_status, sizeof(int));
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "device status read: %s", cudaGetErrorString(err));
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_mx_status, &zero, sizeof(int));
  }
  if (status) *status = v;
  return IPC_OK;
}

}  // namespace ipc
