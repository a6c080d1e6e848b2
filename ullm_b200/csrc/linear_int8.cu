// out[m, n] = (sum_k x[m, k] w[n, k]) * x_scales[m] * w_scales[n] (+ bias[n]) for signed 8-bit x [M, K] and w [N, K] with a 32-bit scale
// per token (row of x) and per channel (row of w); out in float32, bfloat16 or float16.
//
// The sum is a whole number in 32 bits and exact: |sum| <= 2^14 K < 2^31 for K <= 131,071, whatever the order of its terms, so that how
// a product is cut does not show in its result.  The result is formed in float32, times x_scales first, and rounded once.  A token whose
// scale is NaN (a row that had no finite maximum) has NaN results; no other token's change.
//
// Two kernels:
//   linear_int8_tc      the tcgen05 tensor cores (kind::i8), operands by TMA: rows on borders of 16 bytes.  See there.
//   linear_int8_plain   anything else: rows at any address, four products an instruction (dp4a).
#include "tcgen05_util.cuh"

#define LI_MAX_K 131071

struct LiParams {
  const signed char *x, *w;       // (the plain kernel; the other has tensor maps)
  long long x_stride, w_stride;   // bytes between rows
  const float *x_scales, *w_scales;
  const void* bias;               // [N] of out's type, or null
  void* out;                      // [M, N]
  int M, N, K;
  int k_blocks;                   // ceil(K / 128)
  int stages;
  int ksplit;                     // blocks of a cluster that share a tile, each with a range of K
  int* status;
};

template <typename T>
__device__ __forceinline__ T li_result(int sum, float xs, float ws, float bias) {
  return from_f32<T>(fmaf((float)sum * xs, ws, bias));
}

// ---------------------------------------------------------------------------------------------
// Rows at any address: a block makes 32 x 32 results from pieces of 64 k that it packs into words in shared memory.
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) linear_int8_plain(const LiParams p) {
  __shared__ int xs[32][17], ws[32][17];
  pdl_launch_dependents();
  pdl_wait();
  const int n0 = blockIdx.x * 32;
  const long long m0 = (long long)blockIdx.y * 32;
  const int tn = threadIdx.x & 31, tm = threadIdx.x >> 5;  // a thread: column tn, rows tm, tm + 8, ...
  int acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    for (int i = threadIdx.x; i < 32 * 16 * 2; i += 256) {
      const bool of_w = i >= 512;
      const int r = (i >> 4) & 31, q = i & 15, k = k0 + q * 4;
      const long long row = of_w ? n0 + r : m0 + r;
      const signed char* src = (of_w ? p.w + row * p.w_stride : p.x + row * p.x_stride) + k;
      uint32_t v = 0;
      if (row < (of_w ? p.N : p.M)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < p.K) v |= (uint32_t)(unsigned char)src[e] << (8 * e);
      }
      (of_w ? ws : xs)[r][q] = (int)v;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int b = ws[tn][q];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __dp4a(xs[tm + 8 * i][q], b, acc[i]);
    }
    __syncthreads();
  }
  const int n = n0 + tn;
  if (n >= p.N) return;
  const float ws_n = p.w_scales[n], bias = p.bias != nullptr ? to_f32(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + tm + 8 * i;
    if (m < p.M) reinterpret_cast<T*>(p.out)[m * p.N + n] = li_result<T>(acc[i], p.x_scales[m], ws_n, bias);
  }
}

// ---------------------------------------------------------------------------------------------
// The tensor cores.  A tile is 128 channels by NT tokens: channels are the instruction's M (the lanes of tensor memory), tokens its N
// (16 to 256), so that few tokens cost few columns and every weight byte still meets a full instruction.  A block of six warps:
//   warp 0 (one lane)  TMA loads of 128 k of both operands (128-byte swizzle) into a ring of stages;
//   warp 1             tcgen05.mma, 32 k an instruction, the accumulator (32-bit whole numbers) in tensor memory;
//   warps 2 to 5       the end: a thread owns a channel; a warp stores 32 neighbouring channels of a token at a time.
// With few tiles a cluster of `ksplit` blocks shares one, each with a range of K: every block then hands each of the others its sums of
// that block's share of the tokens (distributed shared memory, in the drained ring), and finishes its own share.
// Rows and k outside the operands are read as zeros.
//
// The weights' first stages are asked into L2 before the kernel in front has finished (programmatic dependent launch); nothing is read
// into the block before that: the kernel in front may be the one that makes the weights.
//
// Waits are bounded: one that runs out records ULLM_STATUS_TIMEOUT, the block stores nothing, still meets its cluster, waits (bounded)
// for its own copies in flight, frees its tensor memory and returns.
// ---------------------------------------------------------------------------------------------
#define LI_THREADS 192
#define LI_W_BYTES (128 * 128)
#define LI_MAX_STAGES 12

__device__ __forceinline__ void li_mma(uint32_t lead, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::i8 [%1], %2, %3, %4, p;\n}\n"
      ::"r"(lead), "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void li_tmem_ld16(uint32_t taddr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void li_prefetch(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint32_t li_rank_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void li_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// instruction descriptor of kind::i8: 32-bit sums, signed operands, both K-major
__host__ __device__ constexpr uint32_t li_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <typename T, int NT>
__global__ void __launch_bounds__(LI_THREADS) linear_int8_tc(const __grid_constant__ CUtensorMap w_map,
                                                           const __grid_constant__ CUtensorMap x_map, const LiParams p) {
  constexpr int STAGE = LI_W_BYTES + NT * 128;
  constexpr int TMEM = NT < 32 ? 32 : NT;
  extern __shared__ unsigned char li_smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[LI_MAX_STAGES], empty_bar[LI_MAX_STAGES], acc_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  unsigned char* ring = (unsigned char*)(((uintptr_t)li_smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x % p.ksplit, n0 = (int)blockIdx.x / p.ksplit * 128;
  const int m0 = (int)blockIdx.y * NT;
  const int kb0 = (int)((long long)p.k_blocks * rank / p.ksplit), kb1 = (int)((long long)p.k_blocks * (rank + 1) / p.ksplit);
  const int nkb = kb1 - kb0;  // >= 1: the host splits no further than there are blocks

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&acc_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lin_smem(&tmem_slot)), "r"(TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    pdl_launch_dependents();  // (only now: a kernel behind this one must not hold tensor memory that this one waits for)
  }
  if (warp == 0 && lane < p.stages && lane < nkb) li_prefetch(&w_map, (kb0 + lane) * 128, n0);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_d = tmem_slot;
  pdl_wait();

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t parity = 1;  // a fresh barrier passes a wait on parity 1
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[s], parity)) {
          ullm_report(p.status, ULLM_STATUS_TIMEOUT, 131, kb);
          abort_flag = 1;
          break;
        }
        unsigned char* st = ring + s * STAGE;
        mbar_expect_tx(&full_bar[s], STAGE);
        tma_load_2d(st, &w_map, &full_bar[s], kb * 128, n0);
        tma_load_2d(st + LI_W_BYTES, &x_map, &full_bar[s], kb * 128, m0);
        if (++s == p.stages) s = 0, parity ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = li_idesc(128, NT);
    const uint32_t lead = elect_one();
    const uint64_t desc0 = umma_desc(ring);
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], phase))) {
        if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 132, i);
        abort_flag = 1;
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t a = desc0 + (uint64_t)(s * (STAGE >> 4)), b = a + (LI_W_BYTES >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) li_mma(lead, tmem_d, a + 2 * j, b + 2 * j, idesc, i > 0 || j > 0);  // 32 k: 32 bytes along the row
      umma_commit_warp(lead, lin_smem(&empty_bar[s]));
      if (++s == p.stages) s = 0, phase ^= 1;
    }
    if (ok) umma_commit_warp(lead, lin_smem(&acc_bar));
  }

  // ---- the end ---------------------------------------------------------------------------------
  const int tokens = min(NT, p.M - m0);
  const int quarter = warp & 3, chan = quarter * 32 + lane;  // (warps 2 to 5) this thread's channel of the tile
  const int n = n0 + chan;
  const uint32_t taddr = tmem_d + ((uint32_t)(quarter * 32) << 16);
  T* out = reinterpret_cast<T*>(p.out);
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, mbar_wait(&acc_bar, 0));
    if (!ok) {
      if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 133, 0);
      abort_flag = 1;
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  const float ws = warp >= 2 && n < p.N ? p.w_scales[n] : 0.f;
  const float bias = warp >= 2 && n < p.N && p.bias != nullptr ? to_f32(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
  if (p.ksplit == 1) {
    if (warp >= 2 && ok) {
      for (int c = 0; c < tokens; c += 16) {
        int v[16];
        li_tmem_ld16(taddr + c, v);
        if (n < p.N) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < tokens) out[(size_t)(m0 + c + i) * p.N + n] = li_result<T>(v[i], p.x_scales[m0 + c + i], ws, bias);
        }
      }
    }
  } else {
    const int share = (tokens + p.ksplit - 1) / p.ksplit;  // tokens that a block finishes
    li_cluster_sync();  // every block's ring is drained (its accumulator is complete) or given up
    if (warp >= 2 && ok) {
      for (int c = 0; c < tokens; c += 16) {
        int v[16];
        li_tmem_ld16(taddr + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (c + i >= tokens) break;
          const int to = (c + i) / share, at = (c + i) - to * share;
          const uint32_t dst = li_rank_addr(lin_smem(ring) + (uint32_t)(((rank * share + at) * 128 + chan) * 4), (uint32_t)to);
          asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(dst), "r"(v[i]) : "memory");
        }
      }
    }
    li_cluster_sync();
    if (warp >= 2 && ok && n < p.N) {
      const int* got = reinterpret_cast<const int*>(ring);
      for (int t = 0; t < share && rank * share + t < tokens; ++t) {
        int sum = 0;
        for (int r = 0; r < p.ksplit; ++r) sum += got[(r * share + t) * 128 + chan];
        const int m = m0 + rank * share + t;
        out[(size_t)m * p.N + n] = li_result<T>(sum, p.x_scales[m], ws, bias);
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) {
    // a wait ran out: copies may still be on their way into the ring
    for (int s = 0; s < p.stages && s < nkb; ++s) mbar_wait(&full_bar[s], (((nkb - 1 - s) / p.stages)) & 1);
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_d), "r"(TMEM) : "memory");
  }
}

// rows of 8-bit numbers, boxes of box_rows x 128 bytes
static bool li_map(const void* ptr, long long rows, long long cols, long long stride, int box_rows, CUtensorMap* out) {
  EncodeTiledFn enc = get_encode();
  if (enc == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int g_li_sms = 0;

template <typename T, int NT>
static int li_launch_tc(LiParams p, cudaStream_t st) {
  constexpr int STAGE = LI_W_BYTES + NT * 128;
  constexpr int PER_SM = NT <= 64 ? 2 : 1;
  constexpr int STAGES_MOST = ((PER_SM == 2 ? 110 : 216) * 1024 - 1024) / STAGE;
  constexpr int STAGES = STAGES_MOST < LI_MAX_STAGES ? STAGES_MOST : LI_MAX_STAGES;
  static_assert(STAGES * STAGE >= (NT + 8) * 512, "the ring holds a cluster's sums");
  const int smem = STAGES * STAGE + 1024;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(linear_int8_tc<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return ULLM_ERR_LAUNCH;
    set = true;
  }
  const int n_tiles = (p.N + 127) / 128, m_tiles = (p.M + NT - 1) / NT;
  if (m_tiles > 65535) return ULLM_ERR_UNSUPPORTED;
  const long long tiles = (long long)n_tiles * m_tiles;
  int ksplit = (int)(PER_SM * g_li_sms / tiles);
  if (ksplit > 8) ksplit = 8;
  if (ksplit > p.k_blocks / 2) ksplit = p.k_blocks / 2;
  if (ksplit < 1) ksplit = 1;
  p.ksplit = ksplit;
  p.stages = STAGES;
  CUtensorMap w_map, x_map;
  if (!li_map(p.w, p.N, p.K, p.w_stride, 128, &w_map) || !li_map(p.x, p.M, p.K, p.x_stride, NT, &x_map)) return ULLM_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * ksplit), (unsigned)m_tiles);
  cfg.blockDim = dim3(LI_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ksplit;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_ullm_pdl ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, linear_int8_tc<T, NT>, w_map, x_map, p) != cudaSuccess) {
    cudaGetLastError();
    return ULLM_ERR_LAUNCH;
  }
  return ULLM_OK;
}

template <typename T>
static int li_run(const LiParams& p, cudaStream_t st) {
  const bool aligned = (((uintptr_t)p.x | (uintptr_t)p.w | (uintptr_t)p.x_stride | (uintptr_t)p.w_stride) & 15) == 0;
  if (!aligned) {
    if ((p.M + 31ll) / 32 > 65535) return ULLM_ERR_UNSUPPORTED;
    return ullm_launch_kernel(linear_int8_plain<T>, dim3((p.N + 31) / 32, (p.M + 31) / 32), dim3(256), 0, st, p);
  }
  if (p.M <= 16) return li_launch_tc<T, 16>(p, st);
  if (p.M <= 32) return li_launch_tc<T, 32>(p, st);
  if (p.M <= 64) return li_launch_tc<T, 64>(p, st);
  if (p.M <= 128) return li_launch_tc<T, 128>(p, st);
  return li_launch_tc<T, 256>(p, st);
}

// dtype: of out and bias.  Strides in bytes, at least K.
extern "C" int ullm_linear_int8(int dtype, const void* x, long long x_stride, const void* x_scales, const void* w, long long w_stride,
                                const void* w_scales, const void* bias, void* out, int M, int N, int K, int* status, void* stream) {
  if (M < 0 || N <= 0 || N > (1 << 30) || K <= 0 || K > LI_MAX_K || x_stride < K || w_stride < K) return ULLM_ERR_BAD_SIZE;
  if (dtype != ULLM_DTYPE_F32 && dtype != ULLM_DTYPE_BF16 && dtype != ULLM_DTYPE_F16) return ULLM_ERR_BAD_DTYPE;
  if (M == 0) return ULLM_OK;
  if (g_li_sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&g_li_sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || g_li_sms <= 0)
      return ULLM_ERR_LAUNCH;
  }
  LiParams p = {};
  p.x = (const signed char*)x, p.w = (const signed char*)w, p.x_stride = x_stride, p.w_stride = w_stride;
  p.x_scales = (const float*)x_scales, p.w_scales = (const float*)w_scales, p.bias = bias, p.out = out;
  p.M = M, p.N = N, p.K = K, p.k_blocks = (K + 127) / 128, p.status = status;
  if (dtype == ULLM_DTYPE_F32) return li_run<float>(p, (cudaStream_t)stream);
  if (dtype == ULLM_DTYPE_BF16) return li_run<__nv_bfloat16>(p, (cudaStream_t)stream);
  return li_run<__half>(p, (cudaStream_t)stream);
}
