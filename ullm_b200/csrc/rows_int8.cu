// Rows in 8-bit integers with a 32-bit scale per row, the operands of linear_int8.cu:
//
//   scales[r] = max_c |y[r, c]| / 127,     out[r, c] = the whole number nearest to y[r, c] / scales[r] (ties to even)
//
// of three kinds of rows y, formed in 32-bit and rounded only here:
//   rows as they are                       (a weight's rows, an attention's output)
//   act(gate) * up of rows [gate | up]     (a gated feed-forward)
//   s * rsqrt(mean(s^2) + eps) * w         (RMSNorm) with s = x (+ residual), residual <- round(s)
//
// The norm needs one pass: y = rstd * (s w) with rstd the same for the whole row, so max|y| = rstd max|s w| and the whole numbers are
// those of s w, which the statistics do not enter.  Sum of squares and maximum come out of the same reduction (one barrier).  Rows of any
// size have their scale (squares that 32 bits do not hold: RqSum) as long as s w is finite in 32 bits.
//
// Rounding: s w * (127 / max) + 1.5 * 2^23 in one fused multiply-add leaves the nearest whole number in the sum's low bits (two's
// complement); |s w * (127 / max)| is at most 127 (1 + 2^-23), which is 127 again.  Ties of rows as they are go to even although the
// quotient 127 / max is rounded: v is halfway between two whole numbers where 254 v = odd * max, an odd number below 254, so that 127
// divides that odd number or the significand of max.  The first is v = max / 2, which stands for 63.5 (of 16-bit rows one element in some
// hundred): the quotient is rounded up, and it becomes 64.  Rows of the second kind, one in 127 (bfloat16: none whose quotient is not
// exact), have an exact max / 127, by which the quotient's product is corrected (`rq_quotient`).  All other elements of 16-bit rows are
// further than 2^-19 of their value from a middle, further than the quotient's 2^-23; of 32-bit rows, and of rows that are formed here and
// rounded themselves, what lies nearer to one may go to either side.  A row whose maximum is below 2^-90 is multiplied by 2^100 first, so
// that 127 / max stays finite.
// A row of zeros gets the scale 0 (the norm's formula: NaN where eps is 0 too).  A row that holds an infinity or a NaN has no scale: it
// gets the scale NaN and zeros, so that everything made of it is NaN and the other rows are untouched.  (Between threads the maximum is
// taken of bit patterns, in whose order infinities and then NaN come last.)
//
// The work is bound by memory.  Two forms:
//   rows_int8_kernel   a block takes one row and holds it in registers between the reduction and the store (PER groups of VEC
//                      neighbouring elements per thread, all loads in flight together); rows too long for that are read a second
//                      time.  Norms, few rows, and rows that do not come in pieces of 16 bytes: pieces shifted into place, or element by
//                      element.
//   rows_int8_stream   blocks that stay and take one row after the other, the next rows on their way into shared memory (bulk copies)
//                      while one is worked on.  Many long rows as they are and gated (`rq_choose`); norms never.
#include <type_traits>

#include "tcgen05_util.cuh"

#define RQ_PLAIN 0
#define RQ_ACT 1
#define RQ_NORM 2

struct RqParams {
  const void* x;          // rows of `cols` (RQ_ACT: 2 * cols) elements
  void* residual;         // RQ_NORM: [rows, cols] or null, updated in place
  const float* weight;    // RQ_NORM: [cols]
  signed char* out;       // [rows, cols]
  float* scales;          // [rows]
  long long x_stride, out_stride;  // elements between rows (residual: cols)
  int cols;
  int act;                // RQ_ACT: 0 silu, 1 gelu_tanh
  float eps;
  int rows;
  int* status;
};

// A gate's activation g / (1 + e^-z), z = g (silu) or 2 sqrt(2 / pi) (g + 0.044715 g^3) (gelu_tanh, since (1 + tanh v) / 2 =
// 1 / (1 + e^-2v)), in six instructions without a branch: t = -z log2 e, 2^t, one more, the reciprocal, two products with up's.  Off by
// 2^-22 (|z| + 2.25) of its value: a step or two each, and what the roundings of the exponent make of it.  Where 1 + 2^t passes 2^126 the
// reciprocal is 0, for an activation of up to 2^-119; `rq_act_again` has the rows in which that shows.
__device__ __forceinline__ float rq_exponent(float g, int act) {
  return act == 0 ? g * -1.4426950408889634f : g * fmaf(g * g, -0.10294324f, -2.3022082f);
}
__device__ __forceinline__ float rq_exp2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float rq_gate(float g, float t) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + rq_exp2(t)));
  return g * r;
}
// act(g) * up for any exponent: where 1 is nothing beside 2^t, both factors take half of it (off by 2^-22 (|z| + 3))
__device__ __forceinline__ float rq_gate_times(float g, float up, int act) {
  const float t = rq_exponent(g, act), half = rq_exp2(-0.5f * t);
  return t > 125.f ? (g * half) * (up * half) : rq_gate(g, t) * up;
}
// the largest magnitude, NaN where one is
__device__ __forceinline__ float rq_max(float top, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(v)));
  return r;
}
__device__ __forceinline__ float rq_max(float top, float v, float u) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(fabsf(v)), "f"(fabsf(u)));
  return r;
}
// the larger of top and the VEC magnitudes
template <int VEC>
__device__ __forceinline__ float rq_most(float top, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    top = rq_max(top, v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) top = rq_max(top, v[i], v[i + 1]);
  }
  return top;
}

// (sum, bits of the largest magnitude) over the block, the same in every thread; the order of additions depends on blockDim alone
__device__ __forceinline__ uint32_t rq_reduce(float& sum, float most, bool with_sum, int turn = 0) {
  __shared__ float sums_of[2][32];  // (two sets: one barrier a row)
  __shared__ uint32_t tops_of[2][32];
  float* sums = sums_of[turn];
  uint32_t* tops = tops_of[turn];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
  if (with_sum) sum = warp_sum(sum);
  if (warps == 1) return top;
  if (lane == 0) tops[warp] = top, sums[warp] = sum;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
  if (with_sum) sum = warp_sum(lane < warps ? sums[lane] : 0.f);
  return top;
}

struct RqRow {
  float mul;        // out = round(v * mul)
  uint32_t keep;    // all ones, or 0 for a row that is not finite
  bool tiny;        // ... of v * 2^100
  float step;       // max / 127 (of v * 2^100) where that is exact and `mul` is not, else 0
  float most;       // the row's largest
};
template <typename T, int KIND>
constexpr bool rq_ties = KIND == RQ_PLAIN && !std::is_same<T, __nv_bfloat16>::value;  // whether `step` is asked for at all
template <typename T, int KIND>
__device__ __forceinline__ RqRow rq_row(uint32_t top) {
  RqRow r;
  const float most = r.most = __uint_as_float(top);
  r.tiny = most < 8.077935669463161e-28f;  // 2^-90
  const float top_of = r.tiny ? most * 1.2676506002282294e30f : most;
  float mul = 127.f / top_of;
  const float rest = fmaf(mul, top_of, -127.f);
  if (KIND != RQ_ACT && rest < 0.f) mul = __uint_as_float(__float_as_uint(mul) + 1);
  r.mul = top == 0u ? 0.f : mul;
  r.step = 0.f;
  if constexpr (rq_ties<T, KIND>) {
    const float step = top_of / 127.f;
    if (rest != 0.f && fmaf(step, 127.f, -top_of) == 0.f) r.step = step;
  }
  r.keep = top < 0x7f800000u ? 0xffffffffu : 0u;
  return r;
}
__device__ __forceinline__ float rq_scale(const RqRow& r, float rstd = 1.f, float k = 1.f) {
  return r.keep ? rstd * r.most * k / 127.f : __uint_as_float(0x7fc00000u);
}

// ---- rows that do not come in pieces of 16 bytes (ANY): a thread's group lies on its place of the row, wherever that is in memory ----
// Two neighbouring pieces hold it; a selection of words and a shift bring it into place.
template <typename T>
__device__ __forceinline__ int rq_off(const T* at) {  // elements since the last border of 16 bytes
  return (int)(((uintptr_t)at & 15) / sizeof(T));
}
template <int WORDS>  // w[i] <- the word that lies `bytes` (0 to 15) behind w[i]'s first, i < 4
__device__ __forceinline__ void rq_shift(uint32_t (&w)[WORDS], int bytes) {
  if (bytes & 8) {
#pragma unroll
    for (int i = 0; i + 2 < WORDS; ++i) w[i] = w[i + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int i = 0; i + 1 < WORDS; ++i) w[i] = w[i + 1];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (bytes & 3) * 8);
}
// v <- at[0 .. VEC) of a row that has `left` elements from there on, zeros behind them.  The rows' memory has `before` elements in front of
// `at` and `behind` from there on: pieces that it does not hold whole (at the first row's begin and the last row's end) are not read, but
// their elements one by one.
template <typename T, int VEC>
__device__ __forceinline__ void rq_read(const T* at, long long before, long long behind, int left, float (&v)[VEC]) {
  const int off = rq_off(at);
  if (before >= off && behind >= 2 * VEC - off) {
    const uint4 a = *reinterpret_cast<const uint4*>(at - off), b = *reinterpret_cast<const uint4*>(at - off + VEC);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    rq_shift(w, off * (int)sizeof(T));
    const uint4 u = make_uint4(w[0], w[1], w[2], w[3]);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < left ? to_f32(h[i]) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < left ? to_f32(at[i]) : 0.f;
  }
}
// at[0 .. left) <- v rounded, by a whole warp whose lanes hold neighbouring groups: the piece that a group begins in is stored with the last
// elements of the group in front, where the same warp holds both and the row all of the piece
template <typename T, int VEC>
__device__ __forceinline__ void rq_store_any(T* at, int left, const float (&v)[VEC]) {
  const int off = rq_off(at), lane = threadIdx.x & 31;
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
  uint32_t w[8];
  w[4] = u.x, w[5] = u.y, w[6] = u.z, w[7] = u.w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xffffffffu, w[4 + i], 1);
  // a piece begins `off` elements in front of its group: VEC - off elements into the group before
  const bool mine = lane > 0 && left >= VEC - off, next = lane < 31 && left >= 2 * VEC - off;
  if (off == 0) {
    if (left >= VEC) {
      *reinterpret_cast<uint4*>(at) = u;
      return;
    }
  } else if (mine) {
    rq_shift(w, 16 - off * (int)sizeof(T));
    *reinterpret_cast<uint4*>(at - off) = make_uint4(w[0], w[1], w[2], w[3]);
    if (next) return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < left && (off == 0 || (i < VEC - off ? !mine : !next))) at[i] = e[i];
}

// VEC values of one place of a row; RQ_NORM: unrounded sums in s beside v = s * w
template <typename T, int KIND, int VEC>
__device__ __forceinline__ void rq_load(const RqParams& p, const T* x, const T* res, int c, float (&v)[VEC], float (&s)[VEC]) {
  load_vec<T, VEC>(x + c, v);
  if constexpr (KIND == RQ_ACT) {
    load_vec<T, VEC>(x + p.cols + c, s);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = rq_gate(v[i], rq_exponent(v[i], p.act)) * s[i];
  }
  if constexpr (KIND == RQ_NORM) {
    if (res != nullptr) {
      load_vec<T, VEC>(res + c, s);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] += v[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] = v[i];
    }
    load_vec32<VEC>(p.weight + c, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= s[i];
  }
}
// the same of rows anywhere
template <typename T, int KIND, int VEC>
__device__ __forceinline__ void rq_load_any(const RqParams& p, long long row, const T* x, const T* res, int c, float (&v)[VEC], float (&s)[VEC]) {
  const int left = p.cols - c;
  const long long begin = row * p.x_stride + c, end = (p.rows - 1) * p.x_stride + (KIND == RQ_ACT ? 2ll : 1ll) * p.cols;
  rq_read<T, VEC>(x + c, begin, end - begin, left, v);
  if constexpr (KIND == RQ_ACT) {
    rq_read<T, VEC>(x + p.cols + c, begin + p.cols, end - begin - p.cols, left, s);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = rq_gate(v[i], rq_exponent(v[i], p.act)) * s[i];
  }
  if constexpr (KIND == RQ_NORM) {
    if (res != nullptr) {
      rq_read<T, VEC>(res + c, row * p.cols + c, (p.rows - row) * p.cols - c, left, s);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] += v[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] = v[i];
    }
    if (left >= VEC) {
      load_vec32<VEC>(p.weight + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = i < left ? p.weight[c + i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= s[i];
  }
}
// A thread's sum of the squares of s * k.  Elements beyond 2^64 or so pass what 32 bits hold when they are squared, and where eps is next
// to nothing the smallest fall below it: the sum begins with k = 1 (2^90 for such an eps) and goes on with the next smaller k where it
// reaches 2^100.
struct RqSum {
  float sum = 0.f, k = 1.f;
};
#define RQ_SUM_LIMIT 1.2676506002282294e30f   // 2^100
#define RQ_K_SMALL 1.2379400392853803e27f      // 2^90
#define RQ_K_LARGE 8.271806125530277e-25f      // 2^-80
__device__ __forceinline__ float rq_first_k(float eps) { return eps < 1.0587911840678754e-22f ? RQ_K_SMALL : 1.f; }  // 2^-73
// whether a thread's plain sum of squares has to be formed so
__device__ __forceinline__ bool rq_sum_again(float sum, float eps) { return !(sum < RQ_SUM_LIMIT) || rq_first_k(eps) != 1.f; }
template <int VEC>
__device__ __forceinline__ float rq_squares(const float (&s)[VEC], float sum, float k) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float t = s[i] * k;
    sum = fmaf(t, t, sum);
  }
  return sum;
}
template <int VEC>
__device__ __forceinline__ void rq_add(RqSum& a, const float (&s)[VEC]) {
  float before = a.sum;
  a.sum = rq_squares<VEC>(s, before, a.k);
  if (!(a.sum < RQ_SUM_LIMIT) && a.k > 1.f) {
    before = before / RQ_K_SMALL / RQ_K_SMALL, a.k = 1.f;
    a.sum = rq_squares<VEC>(s, before, a.k);
  }
  if (!(a.sum < RQ_SUM_LIMIT) && a.k == 1.f) {
    before = before * RQ_K_LARGE * RQ_K_LARGE, a.k = RQ_K_LARGE;
    a.sum = rq_squares<VEC>(s, before, a.k);
  }
}
__device__ __forceinline__ void rq_take(RqSum& a, double total, float k) {  // the same of a sum that is there
  if (total * k * k >= RQ_SUM_LIMIT) k = total < RQ_SUM_LIMIT ? 1.f : RQ_K_LARGE;
  a.sum = (float)(total * k * k), a.k = k;
}
template <int KIND, int VEC>
__device__ __forceinline__ void rq_account(const float (&v)[VEC], const float (&s)[VEC], float& sum, float& top) {
  top = rq_most<VEC>(top, v);
  if constexpr (KIND == RQ_NORM) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum = fmaf(s[i], s[i], sum);
  }
}
// (bits of the largest magnitude, the sum of the squares of s * k) over the block; a.k <- that k
template <int KIND>
__device__ __forceinline__ uint32_t rq_join(const RqParams& p, RqSum& a, float most) {
  if constexpr (KIND != RQ_NORM) return rq_reduce(a.sum, most, false);
  float sum = a.k == rq_first_k(p.eps) ? a.sum : __uint_as_float(0x7f800000u);
  const uint32_t top = rq_reduce(sum, most, true);
  if (!(sum < 1.3292279957849159e36f)) {  // 2^120: some thread went on to a smaller k; the smallest is the one that all go by
    float none = 0.f;
    const float k = 1.f / __uint_as_float(rq_reduce(none, 1.f / a.k, false, 1));
    sum = a.sum * (k / a.k) * (k / a.k), a.k = k;
    rq_reduce(sum, 0.f, true);
  }
  a.sum = sum;
  return top;
}
// v / step where `step` is exact: a product with the rounded reciprocal and what it left, so that a quotient of 24 bits comes out as it is
__device__ __forceinline__ float rq_quotient(float v, float mul, float step) {
  const float t = v * mul;
  return fmaf(fmaf(-t, step, v), mul, t);
}
template <bool TIES, int VEC>
__device__ __forceinline__ void rq_store(const RqRow& r, signed char* out, const float (&v)[VEC], int left = VEC) {
  uint32_t q[VEC];
  if (TIES && r.step != 0.f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      q[i] = __float_as_uint(rq_quotient(r.tiny ? v[i] * 1.2676506002282294e30f : v[i], r.mul, r.step) + 12582912.f);
  } else if (r.tiny) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = __float_as_uint(fmaf(v[i] * 1.2676506002282294e30f, r.mul, 12582912.f));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = __float_as_uint(fmaf(v[i], r.mul, 12582912.f));
  }
  if constexpr (VEC % 4 == 0) {
    if (left >= VEC) {
      uint32_t w[VEC / 4];
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i)
        w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410) & r.keep;
      if constexpr (VEC == 8)
        *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
      else
        *reinterpret_cast<uint32_t*>(out) = w[0];
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < left) out[i] = (signed char)(q[i] & r.keep & 0xff);
}

// A gated row in which the elements beyond the fast gate may count, by the whole block, two reads of the row x [gate | up].  They are up to
// 2^-119 |up| each: below half a step, and so nothing, where the row's largest is not below 2^-20 and no up above 2^91.  (Looking for
// such ups would cost every row: 16 x 12,288 2.64 us and 2.80.  Beside one, a gate that far below zero counts as zero.)  Rows of zeros come
// here too: 2,048 x 12,288 of them 52 us, of small rows 65, of others 28.
// (VEC 4 or 1 at a time: with eight the whole kernel would take more than 40 registers, and two blocks of 768 threads no longer find room.)
template <typename T, int VEC>
__device__ __forceinline__ void rq_load_far(const T* x, int cols, int act, int c, float (&v)[VEC]) {
  struct alignas(VEC * sizeof(T)) Piece {
    T e[VEC];
  };
  const Piece g = *reinterpret_cast<const Piece*>(x + c), up = *reinterpret_cast<const Piece*>(x + cols + c);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = rq_gate_times(to_f32(g.e[i]), to_f32(up.e[i]), act);
}
template <typename T, int VEC>
__device__ __noinline__ void rq_act_again(const T* x, signed char* out, float* scale, int cols, int act) {
  float none = 0.f, most = 0.f, v[VEC];
#pragma unroll 1
  for (int c = threadIdx.x * VEC; c < cols; c += blockDim.x * VEC) {
    rq_load_far<T, VEC>(x, cols, act, c, v);
    most = rq_most<VEC>(most, v);
  }
  const RqRow r = rq_row<T, RQ_ACT>(rq_reduce(none, most, false));
  if (threadIdx.x == 0) *scale = rq_scale(r);
#pragma unroll 1
  for (int c = threadIdx.x * VEC; c < cols; c += blockDim.x * VEC) {
    if (r.most == 0.f) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = 0.f;
    } else {
      rq_load_far<T, VEC>(x, cols, act, c, v);
    }
    rq_store<false, VEC>(r, out + c, v);
  }
}
template <int KIND>
__device__ __forceinline__ bool rq_is_far(uint32_t top) {
  return KIND == RQ_ACT && top < 0x35800000u;  // 2^-20
}

// PER > 0: the row in registers, PER * VEC * blockDim >= cols.  PER = 0: any length, read twice.  ANY (with PER > 0): inputs at any address and
// of any length.
template <typename T, int KIND, int VEC, int PER, bool ANY = false>
__global__ void __launch_bounds__(1024) rows_int8_kernel(const RqParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  T* res = KIND == RQ_NORM && p.residual != nullptr ? reinterpret_cast<T*>(p.residual) + row * p.cols : nullptr;
  signed char* out = p.out + row * p.out_stride;
  constexpr int P = PER > 0 ? PER : 1;
  float v[P][VEC], s[P][VEC];
  RqSum sum;
  float most = 0.f;
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) {
        if constexpr (ANY) rq_load_any<T, KIND, VEC>(p, row, x, res, c, v[i], s[i]);
        else rq_load<T, KIND, VEC>(p, x, res, c, v[i], s[i]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = s[i][e] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) rq_account<KIND, VEC>(v[i], s[i], sum.sum, most);
    if constexpr (KIND == RQ_NORM) {
      if (rq_sum_again(sum.sum, p.eps)) {
        sum.sum = 0.f, sum.k = rq_first_k(p.eps);
#pragma unroll
        for (int i = 0; i < PER; ++i) rq_add<VEC>(sum, s[i]);
      }
      if (res != nullptr) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int c = (i * blockDim.x + threadIdx.x) * VEC;
          if constexpr (ANY) rq_store_any<T, VEC>(res + c, p.cols - c, s[i]);  // (whole warps)
          else if (c < p.cols) store_vec<T, VEC>(res + c, s[i]);
        }
      }
    }
  } else {
    double total = 0.0;  // (a thread's share has any number of elements: 2^18 of a row of 2^28)
    for (int c = threadIdx.x * VEC; c < p.cols; c += blockDim.x * VEC) {
      rq_load<T, KIND, VEC>(p, x, res, c, v[0], s[0]);
      float part = 0.f;
      rq_account<KIND, VEC>(v[0], s[0], part, most);
      total += part;
    }
    sum.sum = (float)total;
    if (KIND == RQ_NORM && rq_sum_again(sum.sum, p.eps)) {
      total = 0.0;
      for (int c = threadIdx.x * VEC; c < p.cols; c += blockDim.x * VEC) {
        rq_load<T, KIND, VEC>(p, x, res, c, v[0], s[0]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) total += (double)s[0][i] * s[0][i];
      }
      rq_take(sum, total, rq_first_k(p.eps));
    }
  }
  const uint32_t top = rq_join<KIND>(p, sum, most);
  if constexpr (KIND == RQ_ACT) {
    if (rq_is_far<KIND>(top)) return rq_act_again<T, ANY || VEC < 4 ? 1 : 4>(x, out, p.scales + row, p.cols, p.act);
  }
  const RqRow r = rq_row<T, KIND>(top);
  if (threadIdx.x == 0)
    p.scales[row] = KIND == RQ_NORM ? rq_scale(r, rsqrtf(sum.sum / (float)p.cols + p.eps * sum.k * sum.k), sum.k) : rq_scale(r);
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) rq_store<rq_ties<T, KIND>, VEC>(r, out + c, v[i], ANY ? p.cols - c : VEC);
    }
  } else {
    for (int c = threadIdx.x * VEC; c < p.cols; c += blockDim.x * VEC) {
      rq_load<T, KIND, VEC>(p, x, res, c, v[0], s[0]);
      if (KIND == RQ_NORM && res != nullptr) store_vec<T, VEC>(res + c, s[0]);
      rq_store<rq_ties<T, KIND>, VEC>(r, out + c, v[0]);
    }
  }
}

// One row after the other: two slots of shared memory hold a row's inputs each.  All of a block's threads have read a slot when they meet in
// the reduction, so the copy of a later row into it is asked for right behind it.  Waits are bounded: one that runs out is recorded, and
// the thread goes on without waiting (the block's rows are then wrong, and the status word says so); no copy is asked for behind it, and
// those that are on their way are waited for (bounded) at the end.
#define RQ_SLOTS 2
template <typename T, int KIND>
__global__ void __launch_bounds__(1024) rows_int8_stream(const RqParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), PER = 4;
  extern __shared__ __align__(128) unsigned char rq_ring[];
  __shared__ __align__(8) uint64_t full_bar[RQ_SLOTS];
  const uint32_t bytes = (uint32_t)p.cols * (KIND == RQ_ACT ? 2 : 1) * sizeof(T), slot_bytes = (bytes + 127) & ~127u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < RQ_SLOTS; ++s) mbar_init(&full_bar[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_launch_dependents();
  __syncthreads();
  pdl_wait();
  int asked = 0;  // (thread 0) copies so far, one slot after the other
  auto ask = [&](long long row, int slot) {
    ++asked;
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    mbar_expect_tx(&full_bar[slot], bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     lin_smem(rq_ring + (size_t)slot * slot_bytes)),
                 "l"(x), "r"(bytes), "r"(lin_smem(&full_bar[slot]))
                 : "memory");
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < RQ_SLOTS; ++s)
      if (blockIdx.x + (long long)s * gridDim.x < p.rows) ask(blockIdx.x + (long long)s * gridDim.x, s);
  }
  int slot = 0, turn = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    if (ok && !mbar_wait(&full_bar[slot], parity)) {
      ullm_report(p.status, ULLM_STATUS_TIMEOUT, 138, (int)row);
      ok = false;
    }
    const T* x = reinterpret_cast<const T*>(rq_ring + (size_t)slot * slot_bytes);
    float v[PER][VEC], s[VEC];
    float none = 0.f, most = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) {
        rq_load<T, KIND, VEC>(p, x, nullptr, c, v[i], s);
        most = rq_most<VEC>(most, v[i]);
      }
    }
    const uint32_t top = rq_reduce(none, most, false, turn);
    const RqRow r = rq_row<T, KIND>(top);
    if (threadIdx.x == 0) {
      const long long next = row + (long long)RQ_SLOTS * gridDim.x;
      if (ok && next < p.rows) ask(next, slot);
      p.scales[row] = rq_scale(r);
    }
    signed char* out = p.out + row * p.out_stride;
    if (KIND == RQ_ACT && rq_is_far<KIND>(top)) {
      rq_act_again<T, 4>(reinterpret_cast<const T*>(p.x) + row * p.x_stride, out, p.scales + row, p.cols, p.act);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
        if (c < p.cols) rq_store<rq_ties<T, KIND>, VEC>(r, out + c, v[i]);
      }
    }
    turn ^= 1;
    if (++slot == RQ_SLOTS) slot = 0, parity ^= 1;
  }
  if (!ok && threadIdx.x == 0)  // copies may still be on their way into the slots
    for (int s = 0; s < RQ_SLOTS; ++s) mbar_wait(&full_bar[s], ring_last_parity(s, asked % RQ_SLOTS, ((asked / RQ_SLOTS) & 1) ^ 1));
}

static int g_rq_sms = 0;

// The form that rows take: blocks that stay (`stream`), or a block a row with `per` groups of `vec` elements a thread (0: read twice), at any
// address (`any`).
struct RqForm {
  bool stream, any;
  int vec, per;
};

// Groups of a thread.  One, where a row's groups are threads enough: 2,048 x 4,096 normed 13.0 us, with two 15.2; rows as they are are
// less work and take two from 256 groups on (2,048 x 4,096 6.7 for 8.0, 8 x 8,192 1.61 for 1.69).  Element by element many rows take two
// from 384 on (1,000 x 531 normed 3.3, with one 4.8) and four from 768 (8-bit rows anywhere: 1,000 x 2,043 9.7, with two 11.7, with eight
// 13.3).
static RqForm rq_block_form(int kind, int vec, bool any, int rows, int cols) {
  const int groups = (cols + vec - 1) / vec;
  const int least = vec == 1 ? (rows <= 256 || groups < 384 ? 1 : groups < 768 ? 2 : 4) : kind == RQ_PLAIN && groups >= 256 ? 2 : 1;
  const int per = vec == 1 && groups > 4096 && groups <= 8192 ? 8
                  : groups <= 1024 && least < 2               ? 1
                  : groups <= 2048 && least < 3               ? 2
                  : groups <= 4096                            ? 4
                                                              : 0;
  return {false, any, vec, per};
}

// `wide`: 16-byte pieces of every input row, V bytes of every output row; `borders`: of the weight and the output alone.
static RqForm rq_choose(int kind, int element, int rows, int cols, bool wide, bool borders) {
  const int V = 16 / element, groups = cols / V;
  // Blocks that stay take many and long rows.  us there and below: 2,048 x 25,600 gated 53.7 and 75.7, 2,048 x 16,384 plain 18.8 and 25.9,
  // 1,000 11.7 and 14.3, 300 6.6 and 6.1; 2,048 x 8,192 plain 11.8 and 12.2, gated 19.6 and 19.4.  A norm reads its weight beside the rows
  // and is never faster there (2,048 x 4,096 14.2 and 13.0).
  const long long slot = ((long long)cols * element * (kind == RQ_ACT ? 2 : 1) + 127) / 128 * 128;
  if (kind != RQ_NORM && wide && rows >= 4 * g_rq_sms && groups >= 2048 && groups <= 4096 && RQ_SLOTS * slot <= 208 * 1024)
    return {true, false, V, 4};
  if (wide) return rq_block_form(kind, V, false, rows, cols);
  // Pieces that are shifted into place cost little rows a longer way (the ends' elements come one by one) and many rows less work.  us so
  // and element by element, normed, bfloat16: 1 x 4,091 2.8 and 2.9, 1 x 1,003 2.7 and 1.8; 64 x 2,043 3.0 and 3.0, 300 x 1,003 3.2 and 3.5,
  // 1,000 x 531 5.0 and 3.3, 2,048 x 531 5.8 and 6.4; 2,048 x 4,091 21.4 and 34.4.  Plain 2,048 x 8,001 16.4 and 42.6, gated 2,048 x 9,001
  // 35.6 and 67.2.
  const long long n = (long long)rows * cols;
  const bool many = cols >= 4000 || (cols >= 1000 && n >= 1 << 17) || (cols >= 500 && n >= 1 << 20);
  if (many && borders && cols <= 4096 * V) return rq_block_form(kind, V, true, rows, cols);
  return rq_block_form(kind, 1, false, rows, cols);
}

template <typename T, int KIND>
static int rq_launch_stream(const RqParams& p, int rows, cudaStream_t st) {
  const int groups = p.cols / (16 / (int)sizeof(T)), threads = ((groups + 3) / 4 + 31) / 32 * 32;
  const long long slot = ((long long)p.cols * sizeof(T) * (KIND == RQ_ACT ? 2 : 1) + 127) / 128 * 128;
  const int smem = (int)(RQ_SLOTS * slot);
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(rows_int8_stream<T, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024) != cudaSuccess)
      return ULLM_ERR_LAUNCH;
    set = true;
  }
  int per_sm = 216 * 1024 / (smem + 2048);
  if (per_sm > 1024 / threads) per_sm = 1024 / threads;  // (up to 64 registers a thread)
  if (per_sm < 1) per_sm = 1;
  const int most = per_sm * g_rq_sms, each = (rows + most - 1) / most;  // (every block the same number of rows, or one less)
  return ullm_launch_kernel(rows_int8_stream<T, KIND>, dim3((rows + each - 1) / each), dim3(threads), smem, st, p);
}

template <typename T, int KIND, int VEC, bool ANY>
static int rq_launch_block(const RqParams& p, int rows, int per, cudaStream_t st) {
  const int groups = (p.cols + VEC - 1) / VEC, each = per > 0 ? per : 4, threads = ((groups + each - 1) / each + 31) / 32 * 32;
  auto go = [&](auto kernel) { return ullm_launch_kernel(kernel, dim3(rows), dim3(threads > 1024 ? 1024 : threads), 0, st, p); };
  if (per == 1) return go(rows_int8_kernel<T, KIND, VEC, 1, ANY>);
  if (per == 2) return go(rows_int8_kernel<T, KIND, VEC, 2, ANY>);
  if (per == 4) return go(rows_int8_kernel<T, KIND, VEC, 4, ANY>);
  if constexpr (VEC == 1) {
    if (per == 8) return go(rows_int8_kernel<T, KIND, VEC, 8, ANY>);
  }
  if constexpr (!ANY) return go(rows_int8_kernel<T, KIND, VEC, 0, ANY>);
  return ULLM_ERR_UNSUPPORTED;
}

static bool rq_read_sms() {
  int dev = 0;
  if (g_rq_sms == 0 && (cudaGetDevice(&dev) != cudaSuccess ||
                        cudaDeviceGetAttribute(&g_rq_sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess))
    g_rq_sms = 0;
  return g_rq_sms > 0;
}

template <typename T, int KIND>
static int rq_launch(const RqParams& p, int rows, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool borders = (uintptr_t)p.weight % 16 == 0 && (uintptr_t)p.out % V == 0 && p.out_stride % V == 0;
  const bool wide = borders && p.cols % V == 0 && (uintptr_t)p.x % 16 == 0 && p.x_stride % V == 0 && (uintptr_t)p.residual % 16 == 0;
  if (!rq_read_sms()) return ULLM_ERR_LAUNCH;
  const RqForm f = rq_choose(KIND, sizeof(T), rows, p.cols, wide, borders);
  if constexpr (KIND != RQ_NORM) {
    if (f.stream) return rq_launch_stream<T, KIND>(p, rows, st);
  }
  if (f.any) return rq_launch_block<T, KIND, V, true>(p, rows, f.per, st);
  if (f.vec == V) return rq_launch_block<T, KIND, V, false>(p, rows, f.per, st);
  return rq_launch_block<T, KIND, 1, false>(p, rows, f.per, st);
}

// The form that such rows take: -1 blocks that stay, else 100 * elements of a group + groups of a thread (0: read twice), 1,000 more for rows at
// any address; 0 for sizes that no call takes.  kind: 0 as they are, 1 gated, 2 normed; place: 2 all rows come in pieces of 16 bytes, 1 the
// weight and the output alone lie on borders, 0 nothing does.
extern "C" int ullm_rows_int8_form(int kind, int dtype, int rows, int cols, int place) {
  if (kind < RQ_PLAIN || kind > RQ_NORM || rows <= 0 || cols <= 0 || !rq_read_sms()) return 0;
  const RqForm f = rq_choose(kind, dtype == ULLM_DTYPE_F32 ? 4 : 2, rows, cols, place == 2, place > 0);
  return f.stream ? -1 : 1000 * f.any + 100 * f.vec + f.per;
}

template <int KIND>
static int rq_run(int dtype, RqParams p, int rows, void* stream) {
  if (rows < 0 || p.cols <= 0 || p.cols > (1 << 28) || p.out_stride < p.cols || p.x_stride < p.cols) return ULLM_ERR_BAD_SIZE;
  if (dtype != ULLM_DTYPE_F32 && dtype != ULLM_DTYPE_BF16 && dtype != ULLM_DTYPE_F16) return ULLM_ERR_BAD_DTYPE;
  if (rows == 0) return ULLM_OK;
  cudaStream_t st = (cudaStream_t)stream;
  p.rows = rows;
  if (dtype == ULLM_DTYPE_F32) return rq_launch<float, KIND>(p, rows, st);
  if (dtype == ULLM_DTYPE_BF16) return rq_launch<__nv_bfloat16, KIND>(p, rows, st);
  return rq_launch<__half, KIND>(p, rows, st);
}

// Strides in elements.
extern "C" int ullm_quantize_rows_int8(int dtype, const void* x, long long x_stride, void* out, long long out_stride, void* scales,
                                       int rows, int cols, int* status, void* stream) {
  RqParams p = {};
  p.status = status;
  p.x = x, p.x_stride = x_stride, p.out = (signed char*)out, p.out_stride = out_stride, p.scales = (float*)scales, p.cols = cols;
  return rq_run<RQ_PLAIN>(dtype, p, rows, stream);
}

extern "C" int ullm_act_mul_int8(int dtype, int act, const void* gate_up, void* out, long long out_stride, void* scales, int rows,
                                 int inter, int* status, void* stream) {
  if (act != 0 && act != 1) return ULLM_ERR_BAD_SIZE;
  RqParams p = {};
  p.status = status;
  p.x = gate_up, p.x_stride = 2ll * inter, p.out = (signed char*)out, p.out_stride = out_stride, p.scales = (float*)scales;
  p.cols = inter, p.act = act;
  return rq_run<RQ_ACT>(dtype, p, rows, stream);
}

extern "C" int ullm_add_rmsnorm_int8(int dtype, const void* x, void* residual, const void* weight, void* out, long long out_stride,
                                     void* scales, int rows, int cols, float eps, int* status, void* stream) {
  RqParams p = {};
  p.status = status;
  p.x = x, p.x_stride = cols, p.residual = residual, p.weight = (const float*)weight, p.out = (signed char*)out;
  p.out_stride = out_stride, p.scales = (float*)scales, p.cols = cols, p.eps = eps;
  return rq_run<RQ_NORM>(dtype, p, rows, stream);
}
