// Products with an 8-bit checkpoint for shapes too small for whole 128-row tensor-memory tiles, of any size and
// alignment (16-bit storage):
//   W, WD, G   out [M, K] from sum_b E[m, b] f(x^[k, b])     (weight update, fp32 delta, delta in the storage type)
//   BK         out [K, B] = f'(x^) * sum_m W[m, k] E[m, b]    (error of the layer above)
//
// These are bound by latency, so the aim is one launch, many CTAs and few dependent steps.  A CTA owns a 32 x 64 tile and
// walks the reduction in steps of 64, the next step's operands in registers while mma.sync works on this one's in shared
// memory.  The states are read as codes and f is applied on the way to shared memory: no restored copy, no second launch,
// and where f(x^) does not fit 16 bits, a second operand holds what the first rounds off: the MMAs are idle anyway, and
// the sum then is as accurate as f itself, 2^-20 for sigmoid, silu and gelu, 2^-11 for tanh (tanh.approx: as much as
// fp16's rounding, an eighth of bf16's), instead of a rounding of f as large as the result's own.
// A long reduction with few tiles is split over the CTAs of a cluster, whose partial sums meet in the first CTA's
// shared memory and are added in rank order (deterministic).
#include "ipc_epilogue.cuh"
#include "ipc_generic.cuh"
#include "ipc_mx.cuh"
#include "ipc_ptx.cuh"

namespace ipc {
namespace {

constexpr int SM = 32, SN = 64, SK = 64, STHREADS = 128;
constexpr int S_MAX_SPLIT = 8;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void s_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight elements of a row from column c on, as registers that hold them.  VEC (rows start on 16-byte boundaries and their
// length is a multiple of 8): the vector itself.  Otherwise the two aligned vectors that span them, shifted into
// place when they are used, so that a step's loads do not wait for one another.  A vector that reaches over an end of
// the tensor [base, end) is put together from single elements.
template <bool VEC>
struct Row8 {
  uint4 v[VEC ? 1 : 2];
  uint32_t off;  // byte offset of the first element in v
};
__device__ __forceinline__ uint4 aligned8(uintptr_t at, uintptr_t base, uintptr_t end) {
  if (at >= base && at + 16 <= end) return __ldg(reinterpret_cast<const uint4*>(at));
  uint4 v = make_uint4(0, 0, 0, 0);
  uint16_t* h = reinterpret_cast<uint16_t*>(&v);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at + 2 * j >= base && at + 2 * j + 2 <= end) h[j] = __ldg(reinterpret_cast<const uint16_t*>(at) + j);
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ Row8<VEC> row8(const T* row, int c, int cols, bool in, const T* base, const T* end) {
  Row8<VEC> r;
  r.off = 0;
#pragma unroll
  for (int j = 0; j < (VEC ? 1 : 2); ++j) r.v[j] = make_uint4(0, 0, 0, 0);
  if (!in || c >= cols) return r;
  if constexpr (VEC) {
    r.v[0] = __ldg(reinterpret_cast<const uint4*>(row + c));
  } else {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), lo = at & ~(uintptr_t)15;
    r.off = (uint32_t)(at & 15);
    r.v[0] = aligned8(lo, reinterpret_cast<uintptr_t>(base), reinterpret_cast<uintptr_t>(end));
    if (r.off) r.v[1] = aligned8(lo + 16, reinterpret_cast<uintptr_t>(base), reinterpret_cast<uintptr_t>(end));
  }
  return r;
}
// ... in place; `left`: how many of them belong to the row (the rest become 0)
template <bool VEC>
__device__ __forceinline__ uint4 shifted(const Row8<VEC>& r, int left) {
  if constexpr (VEC) return r.v[0];
  uint32_t w[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w, r.v[VEC ? 0 : 1].x, r.v[VEC ? 0 : 1].y, r.v[VEC ? 0 : 1].z,
                   r.v[VEC ? 0 : 1].w};
#pragma unroll
  for (int j = 0; j < 6; ++j) w[j] = (r.off & 8) ? w[j + 2] : w[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) w[j] = (r.off & 4) ? w[j + 1] : w[j];
  const uint32_t sh = (r.off & 2) * 8;
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[j] = __funnelshift_r(w[j], w[j + 1], sh);
    if (left < 2 * j + 2) o[j] = left > 2 * j ? o[j] & 0xffffu : 0u;
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Whether f(x^) is kept in two parts: relu and identity give c * 2^s, which 16 bits hold (below fp16's smallest normal
// number to within half its smallest step; 2^16, which fp16 states above 65024 read back as, is its infinity).
__host__ __device__ constexpr bool s_low(int act, int mode) {
  return mode != MODE_BK && act != IPC_ACT_RELU && act != IPC_ACT_IDENTITY;
}

// VA, VB: the A operand (E; W for BK) and the E of BK load in whole vectors.
template <typename T, int ACT, int MODE, bool VA, bool VB>
__global__ void __launch_bounds__(STHREADS) mx8_small_kernel(const __grid_constant__ GemmArgs p, int k_per_split) {
  constexpr bool BKM = MODE == MODE_BK;
  constexpr bool LOW = s_low(ACT, MODE);
  constexpr int LDA = BKM ? SM + 8 : SK + 8, LDB = BKM ? SN + 8 : SK + 8;  // shared rows, 16 bytes apart mod 128
  constexpr int ROWS_A = BKM ? SK : SM, ROWS_B = BKM ? SK : SN;
  extern __shared__ __align__(16) uint8_t s_smem[];
  T* sA = reinterpret_cast<T*>(s_smem);
  T* sB = sA + 2 * ROWS_A * LDA;
  T* sL = sB + 2 * ROWS_B * LDB;  // what sB rounds off
  float* red = reinterpret_cast<float*>(sL + (LOW ? 2 * ROWS_B * LDB : 0));
  const int m0 = blockIdx.y * SM, n0 = blockIdx.x * SN;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp >> 1, wn = warp & 1;
  const int C = gridDim.z, rank = blockIdx.z;
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // the first CTA has started
  const int k_lo = rank * k_per_split, k_hi = min(p.Kg, k_lo + k_per_split);
  const T* A = reinterpret_cast<const T*>(p.A);
  const T* E = reinterpret_cast<const T*>(p.Bm);  // BK only

  constexpr int NA = SM * SK / 8 / STHREADS;                       // 16-byte vectors of A a thread moves a step: 2
  constexpr int NB = BKM ? SN * SK / 8 / STHREADS : SN * SK / 16 / STHREADS;  // of E: 4; of codes: 2
  Row8<VA> ra[NA];
  Row8<VB> rbe[BKM ? NB : 1];
  uint4 rb[NB];
  uint32_t rs[NB];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      const int i = tid + STHREADS * j;
      if constexpr (BKM) {  // W rows k0.., columns m0..
        const int r = i / (SM / 8), c = i % (SM / 8) * 8;
        ra[j] = row8<T, VA>(A + (long long)(k0 + r) * p.lda, m0 + c, p.Mg, k0 + r < k_hi, A, A + (long long)p.Kg * p.lda);
      } else {
        const int r = i / (SK / 8), c = i % (SK / 8) * 8;
        ra[j] = row8<T, VA>(A + (long long)(m0 + r) * p.lda, k0 + c, p.Kg, m0 + r < p.Mg, A, A + (long long)p.Mg * p.lda);
      }
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = tid + STHREADS * j;
      if constexpr (BKM) {
        const int r = i / (SN / 8), c = i % (SN / 8) * 8;
        rbe[j] = row8<T, VB>(E + (long long)(k0 + r) * p.ldb, n0 + c, p.Ng, k0 + r < k_hi, E, E + (long long)p.Kg * p.ldb);
      } else {  // 16 codes and their scale byte
        const int r = i / (SK / 16), c = i % (SK / 16) * 16;
        rb[j] = make_uint4(0, 0, 0, 0);
        rs[j] = 0;
        if (n0 + r < p.Ng && k0 + c < p.Kg) {
          rb[j] = __ldg(reinterpret_cast<const uint4*>(p.ck + (long long)(n0 + r) * p.ld_ck + k0 + c));
          rs[j] = p.cks[(long long)((k0 + c) / MX_BLOCK) * p.Ng + n0 + r];
        }
      }
    }
  };
  auto put = [&](int buf, int k0) {
    T* a = sA + buf * ROWS_A * LDA;
    T* b = sB + buf * ROWS_B * LDB;
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      const int i = tid + STHREADS * j;
      const int w = BKM ? SM / 8 : SK / 8;
      // (past a row's end lie the next row's numbers: of no effect in columns that are not stored, zeros for the sum)
      *reinterpret_cast<uint4*>(a + (i / w) * LDA + i % w * 8) = shifted<VA>(ra[j], BKM ? 8 : p.Kg - k0 - i % w * 8);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = tid + STHREADS * j;
      if constexpr (BKM) {
        *reinterpret_cast<uint4*>(b + (i / (SN / 8)) * LDB + i % (SN / 8) * 8) = shifted<VB>(rbe[j], 8);
      } else {
        const int r = i / (SK / 16), c = i % (SK / 16) * 16;
        float q[16];
        mx8_floats(rb[j].x, q);
        mx8_floats(rb[j].y, q + 4);
        mx8_floats(rb[j].z, q + 8);
        mx8_floats(rb[j].w, q + 12);
        const float sc = mx_scale(rs[j]);
        const bool in = n0 + r < p.Ng;
        uint4 o[2], l[2];
        T* h = reinterpret_cast<T*>(o);
        T* lo = reinterpret_cast<T*>(l);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float f = in && k0 + c + e < k_hi ? mx_f<T, ACT>(q[e] * sc) : 0.f;
          // (states up to 2^16 read back from fp16, whose largest number is 65504: the rest goes to the second part)
          constexpr bool OVER = std::is_same<T, __half>::value && (ACT == IPC_ACT_SILU || ACT == IPC_ACT_GELU);
          h[e] = St<T>::st(OVER ? mx_min_nan(f, 65504.f) : f);
          if constexpr (LOW) lo[e] = St<T>::st(f - St<T>::ld(h[e]));
        }
        uint4* dst = reinterpret_cast<uint4*>(b + r * LDB + c);
        dst[0] = o[0];
        dst[1] = o[1];
        if constexpr (LOW) {
          dst = reinterpret_cast<uint4*>(sL + buf * ROWS_B * LDB + r * LDB + c);
          dst[0] = l[0];
          dst[1] = l[1];
        }
      }
    }
  };

  float acc[4][4] = {};
  // BK: the states of this thread's results (two codes at a time, one scale block per warp), read before the sum needs them
  const int gq = lane >> 2, tq = lane & 3;
  uint32_t code2[BKM ? 4 : 1][2], sbyte[2];
  if constexpr (BKM) {
    const int blk = (n0 + wn * 32) / MX_BLOCK;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int m = m0 + wm * 16 + gq + 8 * h;
      const bool in = m < p.Mg && n0 + wn * 32 < p.Ng;  // (a row's codes are padded to whole blocks)
      sbyte[h] = in ? p.cks[(long long)blk * p.Mg + m] : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        code2[j][h] = in ? __ldg(reinterpret_cast<const uint16_t*>(p.ck + (long long)m * p.ld_ck + n0 + wn * 32 + 8 * j + 2 * tq)) : 0u;
    }
  }
  if (k_lo < k_hi) fetch(k_lo);
  int buf = 0;
  for (int k0 = k_lo; k0 < k_hi; k0 += SK, buf ^= 1) {
    put(buf, k0);
    __syncthreads();  // (the other buffer's readers passed the barrier before this one)
    if (k0 + SK < k_hi) fetch(k0 + SK);
    const uint32_t a = saddr(sA + buf * ROWS_A * LDA), b = saddr(sB + buf * ROWS_B * LDB);
    const uint32_t low = saddr(sL + (LOW ? buf * ROWS_B * LDB : 0));
#pragma unroll
    for (int kk = 0; kk < SK; kk += 16) {
      uint32_t fa[4], fb[2][4];
      if constexpr (BKM) {
        // A[m][k] from rows of k: transposed 8x8 blocks (k 0-7, m 0-7), (k 0-7, m 8-15), (k 8-15, m 0-7), ...
        const int kr = kk + (lane & 7) + ((lane & 16) >> 1), mc = wm * 16 + (lane & 8);
        ldsm4t(fa, a + (kr * LDA + mc) * 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // B[k][n]: blocks (k 0-7, n), (k 8-15, n), (k 0-7, n + 8), (k 8-15, n + 8)
          const int br = kk + (lane & 15), bc = wn * 32 + 16 * h + ((lane & 16) >> 1);
          ldsm4t(fb[h], b + (br * LDB + bc) * 2);
        }
      } else {
        const int ar = wm * 16 + (lane & 15), ac = kk + ((lane & 16) >> 1);
        ldsm4(fa, a + (ar * LDA + ac) * 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // rows n: blocks (n 0-7, k 0-7), (n 0-7, k 8-15), (n 8-15, k 0-7), (n 8-15, k 8-15)
          const int br = wn * 32 + 16 * h + (lane & 7) + ((lane & 16) >> 1), bc = kk + (lane & 8);
          ldsm4(fb[h], b + (br * LDB + bc) * 2);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s_mma<T>(acc[j], fa, fb[j >> 1][2 * (j & 1)], fb[j >> 1][2 * (j & 1) + 1]);
      if constexpr (LOW) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          ldsm4(fb[h], low + ((wn * 32 + 16 * h + (lane & 7) + ((lane & 16) >> 1)) * LDB + kk + (lane & 8)) * 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) s_mma<T>(acc[j], fa, fb[j >> 1][2 * (j & 1)], fb[j >> 1][2 * (j & 1) + 1]);
      }
    }
  }

  if (C > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (rank > 0) {  // partial sums to the first CTA, [rank - 1][register][thread]
      const uint32_t dst = mapa0(saddr(red)) + (uint32_t)((rank - 1) * SM * SN + tid) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + (uint32_t)((4 * j + r) * STHREADS * 4)), "f"(acc[j][r])
                       : "memory");
    }
    cluster_sync();
    if (rank > 0) return;
    for (int c = 0; c + 1 < C; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[j][r] += red[c * SM * SN + (4 * j + r) * STHREADS + tid];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + wm * 16 + gq + (r >= 2 ? 8 : 0), n = n0 + wn * 32 + 8 * j + 2 * tq + (r & 1);
      if (m < p.Mg && n < p.Ng) {
        if constexpr (BKM) {
          const float c = (float)(signed char)(code2[j][r >> 1] >> (8 * (r & 1)));
          reinterpret_cast<T*>(p.out)[(long long)m * p.Ng + n] =
              St<T>::st(mx_df_code<T, ACT>(c, mx_scale(sbyte[r >> 1])) * acc[j][r]);
        } else {
          epilogue<T, IPC_ACT_IDENTITY, MODE>(p, 0, m, n, acc[j][r]);
        }
      }
    }
}

template <typename T, int ACT, int MODE, bool VA, bool VB>
int launch_small_t(const GemmArgs& p, cudaStream_t s) {
  constexpr bool BKM = MODE == MODE_BK;
  const long long gx = (p.Ng + SN - 1) / SN, gy = (p.Mg + SM - 1) / SM;
  if (gy > 65535) return set_error(IPC_ERR_ARG, "checkpoint product: %d rows are too many", p.Mg);
  // split the reduction while there are fewer than two CTAs per SM, each part at least two steps long
  const long long steps = (p.Kg + SK - 1) / SK;
  int C = (int)(296 / (gx * gy));
  if (C > steps / 2) C = (int)(steps / 2);
  if (C > S_MAX_SPLIT) C = S_MAX_SPLIT;
  if (C < 1) C = 1;
  const long long per = (steps + C - 1) / C;
  C = steps > 0 ? (int)((steps + per - 1) / per) : 1;
  constexpr int TILES =
      2 * (BKM ? SK * (SM + 8) + SK * (SN + 8) : (SM + SN + (s_low(ACT, MODE) ? SN : 0)) * (SK + 8)) * 2;
  const int smem = TILES + (C - 1) * SM * SN * 4;
  cudaError_t err = ensure_kernel_smem<mx8_small_kernel<T, ACT, MODE, VA, VB>>(TILES + (S_MAX_SPLIT - 1) * SM * SN * 4);
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "checkpoint product smem attribute: %s", cudaGetErrorString(err));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)gx, (unsigned)gy, C);
  cfg.blockDim = dim3(STHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = C;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  err = cudaLaunchKernelEx(&cfg, mx8_small_kernel<T, ACT, MODE, VA, VB>, p, (int)(per * SK));
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "checkpoint product launch: %s", cudaGetErrorString(err));
  count_launch();
  return check_launch("checkpoint product");
}

}  // namespace

int launch_mx8_small(const GemmArgs& p, int mode, int act, int dtype, cudaStream_t s) {
  const bool bk = mode == MODE_BK;
  const bool va = ((reinterpret_cast<uintptr_t>(p.A) | (uintptr_t)(p.lda * 2)) & 15) == 0 && (bk ? p.Mg : p.Kg) % 8 == 0;
  const bool vb = ((reinterpret_cast<uintptr_t>(p.Bm) | (uintptr_t)(p.ldb * 2)) & 15) == 0 && p.Ng % 8 == 0;
  IPC_DISPATCH_DT16(dtype, TT, {
    IPC_DISPATCH_ACT(act, AC, {
      switch (mode) {
        case MODE_W: return va ? launch_small_t<TT, AC, MODE_W, true, true>(p, s) : launch_small_t<TT, AC, MODE_W, false, true>(p, s);
        case MODE_WD: return va ? launch_small_t<TT, AC, MODE_WD, true, true>(p, s) : launch_small_t<TT, AC, MODE_WD, false, true>(p, s);
        case MODE_G: return va ? launch_small_t<TT, AC, MODE_G, true, true>(p, s) : launch_small_t<TT, AC, MODE_G, false, true>(p, s);
        case MODE_BK:
          if (va && vb) return launch_small_t<TT, AC, MODE_BK, true, true>(p, s);
          return va ? launch_small_t<TT, AC, MODE_BK, true, false>(p, s) : launch_small_t<TT, AC, MODE_BK, false, false>(p, s);
        default: return set_error(IPC_ERR_ARG, "checkpoint product: bad mode %d", mode);
      }
    });
  });
  return IPC_OK;
}

}  // namespace ipc
