// out[m, n] = (sum_k x[m, k] w[n, k]) * x_scales[m] * w_scales[n] (+ bias[n]) for signed 8-bit x [M, K] and w [N, K] with a 32-bit scale
// per token (row of x) and per channel (row of w); out in float32, bfloat16 or float16.
//
// The sum is a whole number in 32 bits and exact: |sum| <= 2^14 K < 2^31 for K <= 131,071, whatever the order of its terms, so that how
// a product is cut does not show in its result.  The result is formed in float32, times x_scales first (beyond 2^96 last), and rounded
// once.  A token whose scale is NaN (a row that had no finite maximum) has NaN results; no other token's change.
//
// Three kernels:
//   linear_int8_tc      the tcgen05 tensor cores (kind::i8), operands by TMA (rows on borders of 16 bytes): few tokens, narrow products;
//   linear_int8_pair    the same for many tokens, two SMs to a tile;
//   linear_int8_plain   rows at any address, four products an instruction (dp4a).
// `li_choose` says which of the first two takes a product.
#include <cmath>

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
// A sum times an x_scale beyond 2^96 may pass what 32 bits hold, where the result does not: such tokens meet the other scale first.
__device__ __forceinline__ bool li_large(float xs) { return fabsf(xs) > 7.922816251426434e28f; }

// One channel of W tokens, of which `tokens` exist: out[i * stride] = result of v[i].  All scales are read before the first store,
// which the compiler could not move them in front of (out might be anywhere): 64 columns end in 0.6 us instead of 2.
template <typename T, int W, bool LARGE>
__device__ __forceinline__ void li_store_some(T* out, int stride, const int (&v)[W], const float* xs, float ws, float bias, int tokens) {
  T r[W];
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const float4 s = *reinterpret_cast<const float4*>(xs + i);
    r[i] = li_result<T>(v[i], s.x, ws, bias), r[i + 1] = li_result<T>(v[i + 1], s.y, ws, bias);
    r[i + 2] = li_result<T>(v[i + 2], s.z, ws, bias), r[i + 3] = li_result<T>(v[i + 3], s.w, ws, bias);
    if constexpr (LARGE) {
      const float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (li_large(e[j])) r[i + j] = li_result<T>(v[i + j], ws, e[j], bias);
    }
  }
  if (tokens >= W) {
#pragma unroll
    for (int i = 0; i < W; ++i, out += stride) *out = r[i];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i, out += stride)
      if (i < tokens) *out = r[i];
  }
}

template <typename T, int W>
__device__ __forceinline__ void li_store(bool large, T* out, int stride, const int (&v)[W], const float* xs, float ws, float bias, int tokens) {
  if (large) li_store_some<T, W, true>(out, stride, v, xs, ws, bias, tokens);
  else li_store_some<T, W, false>(out, stride, v, xs, ws, bias, tokens);
}
// The meeting of the 128 finishing threads (barrier 1): whether one of them says so.
__device__ __forceinline__ bool li_meet(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(any)
      : "r"((uint32_t)mine)
      : "memory");
  return any != 0;
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
  const int tn = threadIdx.x & 31, tm = threadIdx.x >> 5;  // a thread: column tn, rows tm, tm + 8, ...
  const int n = n0 + tn;
  const float ws_n = n < p.N ? p.w_scales[n] : 0.f, bias = n < p.N && p.bias != nullptr ? to_f32(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
  for (long long m0 = (long long)blockIdx.y * 32; m0 < p.M; m0 += (long long)gridDim.y * 32) {
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
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long m = m0 + tm + 8 * i;
      if (m < p.M && n < p.N) {
        const float xs_m = p.x_scales[m];
        const bool large = li_large(xs_m);
        reinterpret_cast<T*>(p.out)[m * p.N + n] = li_result<T>(acc[i], large ? ws_n : xs_m, large ? xs_m : ws_n, bias);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// The tensor cores.  A tile is 128 channels by NT tokens: channels are the instruction's M (the lanes of tensor memory), tokens its N
// (16 to 128), so that few tokens cost few columns and every weight byte still meets a full instruction.  A block of six warps:
//   warp 0             TMA loads of both operands (128-byte swizzle) into a ring of stages, KB blocks of 128 k each;
//   warp 1             tcgen05.mma, 32 k an instruction, the accumulator (32-bit whole numbers) in tensor memory;
//   warps 2 to 5       the end: a thread owns a channel; a warp stores 32 neighbouring channels of a token at a time.
// With few tiles a cluster of `ksplit` blocks shares one, each with a range of K: every block then hands each of the others its sums of
// that block's share of the tokens (distributed shared memory, in the drained ring), and finishes its own share.
// Rows and k outside the operands are read as zeros.
//
// The weights' first stages are asked into L2 before the kernel in front has finished (programmatic dependent launch); nothing is read
// into the block before that: the kernel in front may be the one that makes the weights.
//
// Waits for a barrier in shared memory are bounded: one that runs out records ULLM_STATUS_TIMEOUT, the block stores none of the results that
// it waited for (of a shared tile none of the blocks does: the others are told between the cluster's two meetings), waits (bounded) for
// its own copies in flight, frees its tensor memory and returns.  A cluster's meetings and the allocation of tensor memory have no limit of
// their own: they end because every block comes to its meetings and to its release, whatever its waits did.
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

// The copies are asked for by a whole warp, one lane's predicate before the instructions: addresses then stay in uniform registers.  By one
// lane in a branch of its own a stage of 128 k took 0.25 us to ask for, whatever its size, so 0.15.
__device__ __forceinline__ void li_expect(uint32_t lead, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;\n}\n"
      ::"r"(lead), "r"(bar), "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void li_load(uint32_t lead, uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n"
      " @q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];\n}\n"
      ::"r"(lead), "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

// instruction descriptor of kind::i8: 32-bit sums, signed operands, both K-major
__host__ __device__ constexpr uint32_t li_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <typename T, int NT, int KB>
__global__ void __launch_bounds__(LI_THREADS) linear_int8_tc(const __grid_constant__ CUtensorMap w_map,
                                                           const __grid_constant__ CUtensorMap x_map, const LiParams p) {
  constexpr int BLOCK = LI_W_BYTES + NT * 128, STAGE = KB * BLOCK;  // 128 k of both operands; a stage
  constexpr int TMEM = NT < 32 ? 32 : NT;
  extern __shared__ unsigned char li_smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[LI_MAX_STAGES], empty_bar[LI_MAX_STAGES], acc_bar;
  __shared__ uint32_t tmem_slot, next_parity;
  __shared__ int abort_flag, next_stage;  // (next_stage, next_parity: where the loads ended)
  __shared__ __align__(16) float xs_s[NT + 32];  // the tile's token scales
  unsigned char* ring = (unsigned char*)(((uintptr_t)li_smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x % p.ksplit, n0 = (int)blockIdx.x / p.ksplit * 128;
  const int m0 = (int)blockIdx.y * NT;
  const int all = (p.k_blocks + KB - 1) / KB;  // stages of the whole k; this block's are st0 .. st0 + nst - 1, at least one
  const int st0 = (int)((long long)all * rank / p.ksplit), nst = (int)((long long)all * (rank + 1) / p.ksplit) - st0;

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
  if (warp == 0 && lane < p.stages * KB && lane < nst * KB) li_prefetch(&w_map, (st0 * KB + lane) * 128, n0);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_d = tmem_slot;
  pdl_wait();

  bool ok = true;
  if (warp == 0) {
    const uint32_t lead = elect_one();
    const uint32_t ring0 = lin_smem(ring), full0 = lin_smem(&full_bar[0]), empty0 = lin_smem(&empty_bar[0]);
    int s = 0, x = st0 * KB * 128;
    uint32_t parity = 1;  // a fresh barrier passes a wait on parity 1
    for (int i = 0; i < nst; ++i, x += KB * 128) {
      if (!__all_sync(0xffffffffu, mbar_wait_addr(empty0 + s * 8, parity))) {
        if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 131, i);
        abort_flag = 1;
        break;
      }
      const uint32_t st = ring0 + s * STAGE, bar = full0 + s * 8;
      li_expect(lead, bar, STAGE);
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        li_load(lead, st + b * BLOCK, &w_map, bar, x + b * 128, n0);
        li_load(lead, st + b * BLOCK + LI_W_BYTES, &x_map, bar, x + b * 128, m0);
      }
      if (++s == p.stages) s = 0, parity ^= 1;
    }
    if (lane == 0) next_stage = s, next_parity = parity;
  } else if (warp == 1) {
    constexpr uint32_t idesc = li_idesc(128, NT);
    const uint32_t lead = elect_one();
    const uint64_t desc0 = umma_desc(ring);
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nst; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], phase))) {
        if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 132, i);
        abort_flag = 1;
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int j = 0; j < 4 * KB; ++j) {  // 32 k: 32 bytes along the row
        const uint64_t a = desc0 + (uint64_t)(s * (STAGE >> 4) + j / 4 * (BLOCK >> 4) + j % 4 * 2);
        li_mma(lead, tmem_d, a, a + (LI_W_BYTES >> 4), idesc, i > 0 || j > 0);
      }
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
  const float ws = warp >= 2 && n < p.N ? p.w_scales[n] : 0.f;
  const float bias = warp >= 2 && n < p.N && p.bias != nullptr ? to_f32(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
  bool large = false;  // whether one of the tile's tokens is
  if (warp >= 2) {
    for (int i = threadIdx.x - 64; i < tokens; i += 128) {
      const float xs = xs_s[i] = p.x_scales[m0 + i];
      large |= li_large(xs);
    }
    large = li_meet(large);
    ok = __all_sync(0xffffffffu, mbar_wait(&acc_bar, 0));
    if (!ok) {
      if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 133, 0);
      abort_flag = 1;
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  if (p.ksplit == 1) {
    if (warp >= 2 && ok) {
      for (int c = 0; c < tokens; c += 16) {
        int v[16];
        li_tmem_ld16(taddr + c, v);
        if (n < p.N) li_store<T, 16>(large, out + (size_t)(m0 + c) * p.N + n, p.N, v, xs_s + c, ws, bias, tokens - c);
      }
    }
  } else {
    // tokens that a block finishes, a multiple of 4: the sums travel as [block they come from][quad of tokens][channel][4 tokens]
    const int share = ((tokens + p.ksplit - 1) / p.ksplit + 3) & ~3;
    li_cluster_sync();  // every block's ring is drained (its accumulator is complete) or given up
    if (warp == 2 && abort_flag && lane < p.ksplit)
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(li_rank_addr(lin_smem(&abort_flag), lane)), "r"(1) : "memory");
    if (warp >= 2 && ok) {
      const uint32_t mine = lin_smem(ring) + (uint32_t)((rank * (share >> 2)) * 128 + chan) * 16;
      int to = 0, at = 0;  // the block that the next quad goes to, the quad's place there
      uint32_t dst = li_rank_addr(mine, 0);
      for (int c = 0; c < tokens; c += 16) {
        int v[16];
        li_tmem_ld16(taddr + c, v);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          if (c + i < tokens)
            asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)at * 2048u), "r"(v[i]), "r"(v[i + 1]),
                         "r"(v[i + 2]), "r"(v[i + 3])
                         : "memory");
          if (++at == share >> 2) at = 0, dst = li_rank_addr(mine, (uint32_t)min(++to, p.ksplit - 1));
        }
      }
    }
    li_cluster_sync();
    if (warp >= 2 && !abort_flag && n < p.N) {  // (set in any block of the cluster: some of the sums are missing)
      constexpr int W = NT < 32 ? 4 : 16;  // tokens at a time: their loads run beside one another
      const int4* got = reinterpret_cast<const int4*>(ring) + chan;
      const int mine_end = min(share, tokens - rank * share);
      for (int t = 0; t < mine_end; t += W) {
        int v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = 0;
        for (int r = 0; r < p.ksplit; ++r) {
#pragma unroll
          for (int i = 0; i < W; i += 4) {
            if (t + i >= share) break;
            const int4 q = got[(r * (share >> 2) + ((t + i) >> 2)) * 128];
            v[i] += q.x, v[i + 1] += q.y, v[i + 2] += q.z, v[i + 3] += q.w;
          }
        }
        const int m = rank * share + t;
        li_store<T, W>(large, out + (size_t)(m0 + m) * p.N + n, p.N, v, xs_s + m, ws, bias, mine_end - t);
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) {
    // a wait ran out: copies may still be on their way into the ring
    for (int s = 0; s < p.stages; ++s) mbar_wait(&full_bar[s], ring_last_parity(s, next_stage, next_parity));
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_d), "r"(TMEM) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------
// Many tokens.  Two blocks (a cluster of two SMs of one pair, cta_group::2) make tiles of 256 channels by BN tokens: each holds 128 of
// the channels and half of the tokens in shared memory, the leader's instructions read both halves, and each block's tensor memory
// takes its own 128 channels.  With 256 tokens a block loads 32 KB for the work that takes 48 KB alone, which is what keeps the tensor
// cores fed from L2.  Persistent: tiles go round the clusters, tokens fastest (the weights then come from memory once), and two
// accumulators let a tile's end run beside the next one's products.  Tiles of 128 and 192 tokens are for products whose tiles of 256 would
// leave SMs idle in the last round, or take one round more: a round of 74 tiles costs 11.0 us at k = 4,096 with 256 tokens, 7.2 with 192.
//
// Barriers: a stage is full when the bytes of both blocks have come (the leader's barrier counts them all); an instruction group's
// commit frees the stage in both blocks, and tells both that an accumulator is complete; the eight finishing warps of both tell the
// leader that it is drained.
// ---------------------------------------------------------------------------------------------
constexpr int li_pair_stage(int tokens) { return LI_W_BYTES + tokens / 2 * 128; }
constexpr int li_pair_stages(int tokens) { return 200 * 1024 / li_pair_stage(tokens); }  // (8, 7, 6)

__device__ __forceinline__ void li_pair_load(uint32_t lead, uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n"
      " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];\n}\n"
      ::"r"(lead), "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void li_pair_mma(uint32_t lead, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.mma.cta_group::2.kind::i8 [%1], %2, %3, %4, p;\n}\n"
      ::"r"(lead), "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// arrives at the barrier of this address in both blocks when the instructions so far are done
__device__ __forceinline__ void li_pair_commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n .reg .b16 both;\n setp.ne.b32 q, %0, 0;\n mov.b16 both, 3;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%1], both;\n}\n"
      ::"r"(lead), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void li_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool li_wait_cluster(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(lin_smem(bar)), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void li_tmem_ld32(uint32_t taddr, int (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LI_THREADS)
linear_int8_pair(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const LiParams p) {
  constexpr int STAGE = li_pair_stage(BN), STAGES = li_pair_stages(BN), COLUMNS = BN > 128 ? 512 : 256;
  extern __shared__ unsigned char li_smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, go[2], ended, other_ended;  // (where this block's loads ended; where the other's did, if it gave up)
  __shared__ __align__(16) float xs_s[2][BN];  // the token scales of a tile
  unsigned char* ring = (unsigned char*)(((uintptr_t)li_smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x & 1, cluster = (int)blockIdx.x >> 1, clusters = (int)gridDim.x >> 1;
  const int t_tiles = (p.M + BN - 1) / BN;
  const long long tiles = (long long)t_tiles * ((p.N + 255) / 256);

  if (threadIdx.x == 0) {
    abort_flag = 0, other_ended = -1;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  li_cluster_sync();  // the other block runs and its barriers exist
  // Allocating for a pair takes both blocks: what one asks of the other's SM is lost for good where that block has not started yet, or
  // has ended.  So it stands behind the cluster's first meeting, and giving back in front of its last one.
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lin_smem(&tmem_slot)), "r"(COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    pdl_launch_dependents();  // (only now: a kernel behind this one must not hold tensor memory that this one waits for)
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_d = tmem_slot;
  pdl_wait();

  if (warp == 0) {
    const uint32_t lead = elect_one(), both = rank == 0 ? lead : 0u;
    const uint32_t ring0 = lin_smem(ring), full0 = li_rank_addr(lin_smem(&full_bar[0]), 0), own0 = lin_smem(&full_bar[0]);
    const uint32_t empty0 = lin_smem(&empty_bar[0]);
    int s = 0;
    uint32_t parity = 1;  // a fresh barrier passes a wait on parity 1
    bool ok = true;
    for (long long tile = cluster; tile < tiles && ok; tile += clusters) {
      const int c0 = (int)(tile / t_tiles) * 256 + rank * 128, t0 = (int)(tile % t_tiles) * BN + rank * (BN / 2);
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait_addr(empty0 + s * 8, parity))) {
          if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 134, kb);
          abort_flag = 1;
          ok = false;
          break;
        }
        const uint32_t st = ring0 + s * STAGE, bar = full0 + s * 8;
        li_expect(both, own0 + s * 8, 2 * STAGE);  // (the leader's barrier counts both blocks' bytes)
        li_pair_load(lead, st, &w_map, bar, kb * 128, c0);
        li_pair_load(lead, st + LI_W_BYTES, &x_map, bar, kb * 128, t0);
        if (++s == STAGES) s = 0, parity ^= 1;
      }
    }
    if (lane == 0) ended = 2 * s + (int)parity;
    // (the commits that free the last stages arrive in both blocks: neither ends before)
    for (int i = 0; i < STAGES && ok; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_addr(empty0 + s * 8, parity))) {
        if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 139, i);
        abort_flag = 1;
        ok = false;
      }
      if (++s == STAGES) s = 0, parity ^= 1;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = li_idesc(256, BN);
      const uint32_t lead = elect_one();
      const uint64_t desc0 = umma_desc(ring);
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long tile = cluster; tile < tiles && ok; tile += clusters, ++it) {
        const int buf = it & 1;
        if (!__all_sync(0xffffffffu, li_wait_cluster(&acc_empty[buf], ((it >> 1) & 1) ^ 1))) {
          if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 135, it);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem_d + (uint32_t)(buf * BN);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], phase))) {
            if (lane == 0) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 136, kb);
            abort_flag = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t a = desc0 + (uint64_t)(s * (STAGE >> 4)), b = a + (LI_W_BYTES >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) li_pair_mma(lead, d, a + 2 * j, b + 2 * j, idesc, kb > 0 || j > 0);
          li_pair_commit(lead, lin_smem(&empty_bar[s]));
          if (++s == STAGES) s = 0, phase ^= 1;
        }
        if (ok) li_pair_commit(lead, lin_smem(&acc_full[buf]));
      }
    }
  } else {
    const int quarter = warp & 3;
    int it = 0;
    for (long long tile = cluster; tile < tiles; tile += clusters, ++it) {
      const int buf = it & 1;
      const int n = (int)(tile / t_tiles) * 256 + rank * 128 + quarter * 32 + lane, m0 = (int)(tile % t_tiles) * BN;
      const int tokens = min(BN, p.M - m0);
      bool large = false;  // whether one of the tile's tokens is
      for (int i = threadIdx.x - 64; i < BN; i += 128) {
        const float xs = xs_s[buf][i] = i < tokens ? p.x_scales[m0 + i] : 0.f;
        large |= li_large(xs);
      }
      const float ws = n < p.N ? p.w_scales[n] : 0.f;
      const float bias = n < p.N && p.bias != nullptr ? to_f32(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
      // one thread waits (bounded) and tells the others, so that all 128 take the same way out
      if (threadIdx.x == 64) {
        const bool got = mbar_wait(&acc_full[buf], (it >> 1) & 1);
        if (!got) ullm_report(p.status, ULLM_STATUS_TIMEOUT, 137, it), abort_flag = 1;
        go[buf] = got;
      }
      large = li_meet(large);
      if (!go[buf]) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t taddr = tmem_d + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN);
      T* out = reinterpret_cast<T*>(p.out) + (size_t)m0 * p.N + n;
      for (int c = 0; c < tokens; c += 32) {
        int v[32];
        li_tmem_ld32(taddr + c, v);
        if (n < p.N) li_store<T, 32>(large, out + (size_t)c * p.N, p.N, v, xs_s[buf] + c, ws, bias, tokens - c);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) li_arrive_at(li_rank_addr(lin_smem(&acc_empty[buf]), 0));
    }
  }
  __syncthreads();
  if (abort_flag && rank == 1 && threadIdx.x == 0)
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(li_rank_addr(lin_smem(&other_ended), 0)), "r"(ended) : "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  li_cluster_sync();  // nobody arrives at this block's barriers any more, or reads its ring
  if (rank == 0 && threadIdx.x == 0 && (abort_flag || other_ended >= 0)) {
    // A wait ran out: copies may still be on their way into either block's ring, whose bytes the leader's barriers count.  A stage that
    // one block alone has filled never completes: the first such wait runs out, and the rest of that block's copies are there by then.
    const long long all = tiles > cluster ? ((tiles - 1 - cluster) / clusters + 1) * p.k_blocks : 0;
    const int planned = 2 * (int)(all % STAGES) + (int)((all / STAGES) & 1 ^ 1);
    bool more = true;
    for (int s = 0; s < STAGES && more; ++s) more = mbar_wait(&full_bar[s], ring_last_parity(s, ended >> 1, ended & 1));
    const int other = other_ended >= 0 ? other_ended : planned;
    for (int s = 0; s < STAGES && more; ++s) more = mbar_wait(&full_bar[s], ring_last_parity(s, other >> 1, other & 1));
  }
  __syncwarp();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_d), "r"(COLUMNS) : "memory");
  }
  li_cluster_sync();  // (see the allocation)
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

// Whether a product of `tiles` tiles shared by `ks` blocks each has an SM for every block, which then takes a ring of the SM's whole shared
// memory; the others take half of it, two to an SM.  A GPC's SMs are no multiple of a cluster: 32 clusters of 4 find room at once, 34
// take a second round (96 x 2,057 x 1,104 in 8.6 us for 5.4).
static bool li_deep(long long tiles, int ks) {
  return tiles <= (ks == 1 ? g_li_sms : ks == 2 ? g_li_sms * 36 / 74 : ks == 4 ? g_li_sms * 16 / 74 : 0);
}

// Which form a product takes: the one that this estimate finds fastest, in ns.  A launch and a tile's end take `start`; a stage of 128 k
// takes `deep` in a block that has an SM and its ring to itself, else `half`, or `two` for two blocks of an SM; weights come from memory
// at 6.6 GB a ms, partly beside that.  Sharing tiles costs two meetings of the cluster and the way of the sums.  The constants are fitted
// to 280 products (1 to 2,048 tokens, 320 to 24,576 channels, k of 512 to 12,288), each timed in every form: the form chosen here takes
// 0.5 % more than the fastest one on average, 12 % at most, and the estimate is 12 % off on average.  What the forms are for, in us
// beside the nearest other:
//   16, 32, 64 tokens a tile   few tokens: 1 x 6,144 x 4,096 7.0 (shared by two 7.6), 64 x 6,144 x 4,096 8.6 (9.2)
//   shared tiles               few tiles: 8 x 4,096 x 12,288 10.8 (alone 14.3), 16 x 512 x 12,288 5.4 (12.3), 64 x 4,096 x 12,288 12.5 (18.1)
//   128 tokens a tile          96 x 24,576 x 4,096 22.5 (64 tokens 30.6, pairs 24); 512 x 4,096 x 4,096 10.4 (pairs 11.0)
//   pairs, 128 tokens          256 x 24,576 x 4,096 27.1 (128 alone 37, 256 in pairs 29.8)
//   pairs, 192 tokens          512 x 6,144 x 4,096 13.5 (128 in pairs 16.4); 768 x 4,096 x 12,288 28.0 (256 in pairs 34.8)
//   pairs, 256 tokens          512 x 24,576 x 4,096 38.5 (192 tokens 41, 128 alone 64); 2,048 x 24,576 x 4,096 126 (133, 235)
struct LiForm {
  int pair, tile, ksplit;
};
static LiForm li_choose(int M, int N, int K) {
  static const int tile[4] = {16, 32, 64, 128}, start[4] = {1930, 2250, 2900, 3200}, deep[4] = {101, 112, 157, 204},
                   half[4] = {152, 200, 348, 276}, two[4] = {291, 287, 348, 456};
  static const int pair_tile[3] = {128, 192, 256}, pair_start[3] = {5210, 4030, 4470}, pair_block[3] = {182, 257, 293};
  const int k_blocks = (K + 127) / 128;
  const long long sms = g_li_sms;
  const double weights = (double)N * K;
  LiForm best = {0, 16, 1};
  double least = 1e300;
  for (int i = 0; i < 4; ++i) {
    const int nt = tile[i], kb = nt < 64 ? 2 : 1;  // (blocks of k a stage)
    if ((i > 0 && nt >= 2ll * M) || (nt < 64 && nt < M) || (M - 1) / nt >= 65535) continue;  // (a grid has 65,535 rows; pairs go round)
    const long long tiles = (long long)((N + 127) / 128) * ((M + nt - 1) / nt);
    for (int ks = 1; ks <= 8; ks *= 2) {
      const bool own = li_deep(tiles, ks);
      if (ks > 1 && (k_blocks < 2 * ks || (!own && (nt >= 64 || ks < 8 || tiles * ks > sms)))) continue;
      const long long rounds = tiles * ks / (2 * sms), rest = tiles * ks % (2 * sms);
      const double stage = own ? deep[i] : (double)rounds * two[i] + (rest == 0 ? 0 : rest <= sms ? half[i] : two[i]);
      const double t = start[i] + hypot(stage * (((k_blocks + kb - 1) / kb + ks - 1) / ks * kb), weights / 6600) +
                       (ks > 1 ? 1200 + 14 * (nt < M ? nt : M) : 0);
      if (t < least) least = t, best = {0, nt, ks};
    }
  }
  for (int i = 0; i < 3 && M > 64; ++i) {
    const long long tiles = (long long)((N + 255) / 256) * ((M + pair_tile[i] - 1) / pair_tile[i]);
    const double t = pair_start[i] + hypot((double)((tiles + sms / 2 - 1) / (sms / 2)) * k_blocks * pair_block[i], weights / 6600);
    if (t < least) least = t, best = {1, pair_tile[i], 1};
  }
  return best;
}

template <typename T, int NT, int KB>
static int li_launch_tc(LiParams p, int ksplit, cudaStream_t st) {
  constexpr int STAGE = KB * (LI_W_BYTES + NT * 128);
  constexpr int DEEP = 216 * 1024 / STAGE < LI_MAX_STAGES ? 216 * 1024 / STAGE : LI_MAX_STAGES, HALF = 109 * 1024 / STAGE;
  static_assert((NT < 64 ? HALF : DEEP) * STAGE >= (NT + 32) * 512, "the ring holds a cluster's sums");
  const int n_tiles = (p.N + 127) / 128, m_tiles = (p.M + NT - 1) / NT;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(linear_int8_tc<T, NT, KB>, cudaFuncAttributeMaxDynamicSharedMemorySize, DEEP * STAGE + 1024) != cudaSuccess)
      return ULLM_ERR_LAUNCH;
    set = true;
  }
  p.ksplit = ksplit;
  p.stages = li_deep((long long)n_tiles * m_tiles, ksplit) ? DEEP : HALF;
  const int smem = p.stages * STAGE + 1024;
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
  if (cudaLaunchKernelEx(&cfg, linear_int8_tc<T, NT, KB>, w_map, x_map, p) != cudaSuccess) {
    cudaGetLastError();
    return ULLM_ERR_LAUNCH;
  }
  return ULLM_OK;
}

template <typename T, int BN>
static int li_launch_pair(const LiParams& p, cudaStream_t st) {
  const int smem = li_pair_stages(BN) * li_pair_stage(BN) + 1024;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(linear_int8_pair<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return ULLM_ERR_LAUNCH;
    set = true;
  }
  const long long tiles = (long long)((p.M + BN - 1) / BN) * ((p.N + 255) / 256);
  const int clusters = (int)(tiles < g_li_sms / 2 ? tiles : g_li_sms / 2);
  CUtensorMap w_map, x_map;
  if (!li_map(p.w, p.N, p.K, p.w_stride, 128, &w_map) || !li_map(p.x, p.M, p.K, p.x_stride, BN / 2, &x_map)) return ULLM_ERR_LAUNCH;
  return ullm_launch_kernel(linear_int8_pair<T, BN>, dim3(2 * clusters), dim3(LI_THREADS), smem, st, w_map, x_map, p);
}

template <typename T>
static int li_run(const LiParams& p, cudaStream_t st) {
  const bool aligned = (((uintptr_t)p.x | (uintptr_t)p.w | (uintptr_t)p.x_stride | (uintptr_t)p.w_stride) & 15) == 0;
  if (!aligned) {
    return ullm_launch_kernel(linear_int8_plain<T>, dim3((p.N + 31) / 32, p.M <= 65535 * 32 ? (p.M + 31) / 32 : 65535), dim3(256), 0, st, p);
  }
  const LiForm f = li_choose(p.M, p.N, p.K);
  if (f.pair && f.tile == 128) return li_launch_pair<T, 128>(p, st);
  if (f.pair && f.tile == 192) return li_launch_pair<T, 192>(p, st);
  if (f.pair) return li_launch_pair<T, 256>(p, st);
  if (f.tile == 16) return li_launch_tc<T, 16, 2>(p, f.ksplit, st);
  if (f.tile == 32) return li_launch_tc<T, 32, 2>(p, f.ksplit, st);
  if (f.tile == 64) return li_launch_tc<T, 64, 1>(p, f.ksplit, st);
  return li_launch_tc<T, 128, 1>(p, f.ksplit, st);
}

static int li_read_sms() {
  int dev = 0;
  if (g_li_sms == 0 && (cudaGetDevice(&dev) != cudaSuccess ||
                        cudaDeviceGetAttribute(&g_li_sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess))
    g_li_sms = 0;
  return g_li_sms;
}

// The kernel that a product of these sizes takes: 1000 * blocks that share a tile + tokens of a tile, negative for pairs of blocks.
extern "C" int ullm_linear_int8_form(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || li_read_sms() <= 0) return 0;
  const LiForm f = li_choose(M, N, K);
  return f.pair ? -f.tile : 1000 * f.ksplit + f.tile;
}

extern "C" int ullm_ring_last_parity(int t, int s, int parity) { return (int)ring_last_parity(t, s, (uint32_t)parity); }

// dtype: of out and bias.  Strides in bytes, at least K.
extern "C" int ullm_linear_int8(int dtype, const void* x, long long x_stride, const void* x_scales, const void* w, long long w_stride,
                                const void* w_scales, const void* bias, void* out, int M, int N, int K, int* status, void* stream) {
  if (M < 0 || M > (1 << 30) || N <= 0 || N > (1 << 30) || K <= 0 || K > LI_MAX_K || x_stride < K || w_stride < K) return ULLM_ERR_BAD_SIZE;
  if (dtype != ULLM_DTYPE_F32 && dtype != ULLM_DTYPE_BF16 && dtype != ULLM_DTYPE_F16) return ULLM_ERR_BAD_DTYPE;
  if (M == 0) return ULLM_OK;
  if (li_read_sms() <= 0) return ULLM_ERR_LAUNCH;
  LiParams p = {};
  p.x = (const signed char*)x, p.w = (const signed char*)w, p.x_stride = x_stride, p.w_stride = w_stride;
  p.x_scales = (const float*)x_scales, p.w_scales = (const float*)w_scales, p.bias = bias, p.out = out;
  p.M = M, p.N = N, p.K = K, p.k_blocks = (K + 127) / 128, p.status = status;
  if (dtype == ULLM_DTYPE_F32) return li_run<float>(p, (cudaStream_t)stream);
  if (dtype == ULLM_DTYPE_BF16) return li_run<__nv_bfloat16>(p, (cudaStream_t)stream);
  return li_run<__half>(p, (cudaStream_t)stream);
}
