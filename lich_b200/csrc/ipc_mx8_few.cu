// Products with an 8-bit checkpoint of a few samples, in fp32 FMAs (f and f' of ipc_mx.cuh in fp32, off by 2^-20 of themselves,
// tanh in 16-bit storage by 2^-11; the result is rounded once):
//   W, WD, G   (up to 16) out[m][k] from sum_b E[m][b] f(x^[k][b]): bound by writing (W: reading and writing) M x K numbers.
//              A CTA takes 64 x 256 of them, with its 256 states' f and its 64 errors' rows in shared memory.
//   BK         (up to 4) out[k][b] = f'(x^[k][b]) sum_m W[m][k] E[m][b]: bound by one read of W.  A CTA takes 64 columns of
//              W, which its warps read along the rows, a row each, eight in flight; the rows are split over the warps and the
//              CTAs of a cluster, whose sums meet in the first CTA's shared memory and are added in a fixed order.
// A tensor-core tile would be all padding here: 4096 x 4096 with one sample took 44 and 40 us in the 64-column tiles of
// mx8_small_kernel, and takes 11 and 17 us; with 16 samples the MMAs win (17 us on tcgen05, 24 us) over 23 and 52.
#include "ipc_epilogue.cuh"
#include "ipc_generic.cuh"
#include "ipc_mx.cuh"
#include "ipc_ptx.cuh"

namespace ipc {
namespace {

constexpr int FEW = 16;
constexpr int OR = 8, OM = 8 * OR, OK = 256, OTHREADS = 256;  // rows of a thread, of a CTA; columns

// ------------------------------------------------------------------------------------- W, WD, G
// VEC: rows of out start on 16-byte boundaries; a thread owns 8 neighbouring columns (else columns lane, lane + 32, ...) of
// 8 rows, so that a sample costs 10 shared-memory wavefronts for 64 FMAs.
template <typename T, int ACT, int MODE, bool VEC>
__global__ void __launch_bounds__(OTHREADS) mx8_outer_kernel(const __grid_constant__ GemmArgs p) {
  using O = typename std::conditional<MODE == MODE_WD, float, T>::type;
  __shared__ __align__(16) float sA[FEW][OK];
  __shared__ __align__(16) float sE[FEW][OM];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int k0 = blockIdx.x * OK, m0 = blockIdx.y * OM, B = p.Kg;
  {
    const int k = k0 + tid;
    if (k < p.Ng) {
      const uint4 c = __ldg(reinterpret_cast<const uint4*>(p.ck + (long long)k * p.ld_ck));
      const float sc = mx_scale(p.cks[k]);
      float v[FEW];
      mx8_floats(c.x, v);
      mx8_floats(c.y, v + 4);
      mx8_floats(c.z, v + 8);
      mx8_floats(c.w, v + 12);
#pragma unroll
      for (int b = 0; b < FEW; ++b)
        if (b < B) sA[b][tid] = mx_f<T, ACT>(v[b] * sc);
    }
  }
  const T* E = reinterpret_cast<const T*>(p.A);
  for (int i = tid; i < OM * FEW; i += OTHREADS) {
    const int r = i / FEW, b = i % FEW;
    if (b < B) sE[b][r] = m0 + r < p.Mg ? St<T>::ld(E[(long long)(m0 + r) * p.lda + b]) : 0.f;
  }
  __syncthreads();
  float acc[OR][8] = {};
  for (int b = 0; b < B; ++b) {
    float a[8];
    if constexpr (VEC) {
      const float4 a0 = *reinterpret_cast<const float4*>(&sA[b][8 * lane]), a1 = *reinterpret_cast<const float4*>(&sA[b][8 * lane + 4]);
      a[0] = a0.x; a[1] = a0.y; a[2] = a0.z; a[3] = a0.w; a[4] = a1.x; a[5] = a1.y; a[6] = a1.z; a[7] = a1.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = sA[b][lane + 32 * j];
    }
    const float4 e0 = *reinterpret_cast<const float4*>(&sE[b][OR * warp]), e1 = *reinterpret_cast<const float4*>(&sE[b][OR * warp + 4]);
    const float e[OR] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
    for (int i = 0; i < OR; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(e[i], a[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < OR; ++i) {
    const int m = m0 + OR * warp + i;
    if (m >= p.Mg) break;
    O* row = reinterpret_cast<O*>(p.out) + (long long)m * p.Ng;
    if constexpr (VEC) {
      const int k = k0 + 8 * lane;
      if (k < p.Ng) {
        constexpr int NV = 8 * (int)sizeof(O) / 16;
        uint4* at = reinterpret_cast<uint4*>(row + k);
        uint4 raw[NV];
        O* h = reinterpret_cast<O*>(raw);
        if (MODE == MODE_W || (MODE == MODE_WD && p.accumulate))
#pragma unroll
          for (int j = 0; j < NV; ++j) raw[j] = at[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = p.scale * acc[i][j];
          if (MODE == MODE_W || (MODE == MODE_WD && p.accumulate)) h[j] = St<O>::st(St<O>::ld(h[j]) + v);
          else h[j] = St<O>::st(v);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) at[j] = raw[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = k0 + lane + 32 * j;
        if (k >= p.Ng) break;
        const float v = p.scale * acc[i][j];
        if (MODE == MODE_W || (MODE == MODE_WD && p.accumulate)) row[k] = St<O>::st(St<O>::ld(row[k]) + v);
        else row[k] = St<O>::st(v);
      }
    }
  }
}

template <typename T, int ACT, int MODE>
int launch_outer_t(const GemmArgs& p, cudaStream_t s) {
  const dim3 grid((p.Ng + OK - 1) / OK, (p.Mg + OM - 1) / OM);
  if (grid.y > 65535u) return set_error(IPC_ERR_ARG, "checkpoint product: %d rows are too many", p.Mg);
  const int size = MODE == MODE_WD ? 4 : (int)sizeof(T);
  const bool vec = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)((long long)p.Ng * size)) & 15) == 0 && p.Ng % 8 == 0;
  if (vec)
    mx8_outer_kernel<T, ACT, MODE, true><<<grid, OTHREADS, 0, s>>>(p);
  else
    mx8_outer_kernel<T, ACT, MODE, false><<<grid, OTHREADS, 0, s>>>(p);
  count_launch();
  return check_launch("checkpoint product of few samples");
}

// -------------------------------------------------------------------------------------------- BK
constexpr int BC = 64;        // columns of W a CTA takes
constexpr int BTHREADS = 256;
constexpr int BU = 8;         // rows of W in flight in a warp
constexpr int BROWS = BU * 8 * 4;  // rows whose E is in shared memory at a time
constexpr int B_SPLIT = 8;

// NB: samples, rounded up to 1 or 4.  A lane owns columns 2 lane, 2 lane + 1 (PAIR: rows start on boundaries of two
// elements) or lane, lane + 32.
template <typename T, int ACT, int NB, bool PAIR>
__global__ void __launch_bounds__(BTHREADS) mx8_columns_kernel(const __grid_constant__ GemmArgs p, int rows_per) {
  extern __shared__ __align__(16) float f_smem[];
  float* red = f_smem;                          // [8 warps][64 columns][NB]
  float* sE = red + 8 * BC * NB;                // [BROWS][NB]
  float* other = sE + BROWS * NB;               // [C - 1][64][NB], in the first CTA
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = blockIdx.x * BC, B = p.Ng, C = gridDim.y, rank = blockIdx.y;
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // the first CTA has started
  const int m_lo = rank * rows_per, m_hi = min(p.Kg, m_lo + rows_per);
  const T* W = reinterpret_cast<const T*>(p.A);
  const T* E = reinterpret_cast<const T*>(p.Bm);
  const int cl[2] = {PAIR ? 2 * lane : lane, PAIR ? 2 * lane + 1 : lane + 32};
  const bool in[2] = {c0 + cl[0] < p.Mg, c0 + cl[1] < p.Mg};
  float acc[2][NB] = {};
  struct alignas(2 * sizeof(T)) Two {
    T v[2];
  };
  Two w[BU];
  auto fetch = [&](int m) {
#pragma unroll
    for (int u = 0; u < BU; ++u) {
      w[u].v[0] = w[u].v[1] = St<T>::st(0.f);
      if (m + u < m_hi) {
        const T* row = W + (long long)(m + u) * p.lda + c0;
        if constexpr (PAIR) {
          if (in[0]) w[u] = *reinterpret_cast<const Two*>(row + 2 * lane);  // (an even number of columns)
        } else {
          if (in[0]) w[u].v[0] = row[cl[0]];
          if (in[1]) w[u].v[1] = row[cl[1]];
        }
      }
    }
  };
  for (int r0 = m_lo; r0 < m_hi; r0 += BROWS) {
    if (r0 + BU * warp < m_hi) fetch(r0 + BU * warp);  // under the staging of E
    __syncthreads();
    for (int i = tid; i < BROWS * NB; i += BTHREADS) {
      const int r = i / NB, b = i % NB;
      sE[i] = (r0 + r < m_hi && b < B) ? St<T>::ld(E[(long long)(r0 + r) * p.ldb + b]) : 0.f;
    }
    __syncthreads();
#pragma unroll 1
    for (int q = BU * warp; q < BROWS && r0 + q < m_hi; q += BU * 8) {
      float x[BU][2];
#pragma unroll
      for (int u = 0; u < BU; ++u) {
        x[u][0] = St<T>::ld(w[u].v[0]);
        x[u][1] = St<T>::ld(w[u].v[1]);
      }
      if (q + BU * 8 < BROWS && r0 + q + BU * 8 < m_hi) fetch(r0 + q + BU * 8);
#pragma unroll
      for (int u = 0; u < BU; ++u) {
        float e[NB];
        if constexpr (NB % 4 == 0) {
#pragma unroll
          for (int b = 0; b < NB; b += 4) *reinterpret_cast<float4*>(e + b) = *reinterpret_cast<const float4*>(sE + (q + u) * NB + b);
        } else {
          e[0] = sE[q + u];
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          acc[0][b] = fmaf(x[u][0], e[b], acc[0][b]);
          acc[1][b] = fmaf(x[u][1], e[b], acc[1][b]);
        }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int b = 0; b < NB; ++b) red[(warp * BC + cl[h]) * NB + b] = acc[h][b];
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  for (int i = tid; i < BC * NB; i += BTHREADS) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += red[w * BC * NB + i];
    if (rank == 0)
      red[i] = sum;
    else
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa0(saddr(other)) + 4u * (uint32_t)((rank - 1) * BC * NB + i)),
                   "f"(sum)
                   : "memory");
  }
  if (C > 1) {
    cluster_sync();
    if (rank > 0) return;
  }
  for (int i = tid; i < BC * NB; i += BTHREADS) {  // (each thread reads back its own sums)
    float sum = red[i];
    for (int c = 0; c + 1 < C; ++c) sum += other[c * BC * NB + i];
    const int k = c0 + i / NB, b = i % NB;
    if (k < p.Mg && b < B) {
      const float f = mx_df_code<T, ACT>((float)p.ck[(long long)k * p.ld_ck + b], mx_scale(p.cks[k]));
      reinterpret_cast<T*>(p.out)[(long long)k * B + b] = St<T>::st(f * sum);
    }
  }
}

template <typename T, int ACT, int NB, bool PAIR>
int launch_columns_t(const GemmArgs& p, cudaStream_t s) {
  const long long gx = (p.Mg + BC - 1) / BC;
  // split the rows while there are fewer than four CTAs per SM, at least a round of every warp's rows in each part
  const long long rounds = (p.Kg + BU * 8 - 1) / (BU * 8);
  int C = (int)(592 / gx);
  if (C > rounds) C = (int)rounds;
  if (C > B_SPLIT) C = B_SPLIT;
  if (C < 1) C = 1;
  const long long per = (rounds + C - 1) / C;
  C = rounds > 0 ? (int)((rounds + per - 1) / per) : 1;
  const int fixed = (8 * BC + BROWS) * NB * 4, smem = fixed + (C - 1) * BC * NB * 4, most = fixed + (B_SPLIT - 1) * BC * NB * 4;
  cudaError_t err = ensure_kernel_smem<mx8_columns_kernel<T, ACT, NB, PAIR>>(most);
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "checkpoint product smem attribute: %s", cudaGetErrorString(err));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)gx, C);
  cfg.blockDim = dim3(BTHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = C;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  err = cudaLaunchKernelEx(&cfg, mx8_columns_kernel<T, ACT, NB, PAIR>, p, (int)(per * BU * 8));
  if (err != cudaSuccess) return set_error(IPC_ERR_CUDA, "checkpoint product launch: %s", cudaGetErrorString(err));
  count_launch();
  return check_launch("checkpoint product of few samples");
}

}  // namespace

int launch_mx8_few(const GemmArgs& p, int mode, int act, int dtype, cudaStream_t s) {
  IPC_DISPATCH_DT(dtype, TT, {
    IPC_DISPATCH_ACT(act, AC, {
      switch (mode) {
        case MODE_W: return launch_outer_t<TT, AC, MODE_W>(p, s);
        case MODE_WD: return launch_outer_t<TT, AC, MODE_WD>(p, s);
        case MODE_G: return launch_outer_t<TT, AC, MODE_G>(p, s);
        case MODE_BK:
          if (p.Mg % 2 == 0 && reinterpret_cast<uintptr_t>(p.A) % (2 * sizeof(TT)) == 0)
            return p.Ng == 1 ? launch_columns_t<TT, AC, 1, true>(p, s) : launch_columns_t<TT, AC, 4, true>(p, s);
          return p.Ng == 1 ? launch_columns_t<TT, AC, 1, false>(p, s) : launch_columns_t<TT, AC, 4, false>(p, s);
        default: return set_error(IPC_ERR_ARG, "checkpoint product: bad mode %d", mode);
      }
    });
  });
  return IPC_OK;
}

}  // namespace ipc
