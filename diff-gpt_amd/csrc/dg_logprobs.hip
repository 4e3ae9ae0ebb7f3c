// Log probabilities of given tokens, entropy and the most likely alternatives
// (dg_token_logprobs): one pass over the logits.
//
// A wavefront takes a row.  The softmax keeps, per lane, a running maximum m, the sum s of
// e^(x - m) and the sum t of (x - m) e^(x - m); raising m by d turns t into
// e^-d (t - d s).  Then log p(id) = x[id] - m - log s and the entropy is log s - t / s.
#include "dg_common.h"

namespace dg {

struct LogprobArgs {
  const void* x;
  int64_t ld, M, V;
  const int64_t* ids;
  void* logprob;
  void* entropy;
  int top;
  void* top_logprob;
  int64_t* top_ids;
};

template <typename T>
struct LpAcc {
  using type = float;
  static __device__ __forceinline__ float load(T x) { return to_f32(x); }
  static __device__ __forceinline__ float exp(float x) { return __expf(x); }
  static __device__ __forceinline__ float log(float x) { return logf(x); }
};
template <>
struct LpAcc<double> {
  using type = double;
  static __device__ __forceinline__ double load(double x) { return x; }
  static __device__ __forceinline__ double exp(double x) { return ::exp(x); }
  static __device__ __forceinline__ double log(double x) { return ::log(x); }
};

// m, s, t of a part of the row, joined with another part's
template <typename S, typename A>
__device__ __forceinline__ void join_part(A& m, A& s, A& t, A m2, A s2, A t2) {
  const A ninf = -(A)__builtin_huge_valf();
  const A mn = m > m2 ? m : m2;
  if (mn == ninf) {  // neither holds a probability; a NaN stays in s
    s += s2;
    return;
  }
  // a part at -inf has s = 0 (or NaN) and no t; one whose factor vanishes, the difference
  // of two finite logits may overflow, adds nothing
  const A d1 = m - mn, d2 = m2 - mn;
  const A f1 = S::exp(d1), f2 = S::exp(d2);
  t = (f1 == (A)0 ? (A)0 : f1 * (t + d1 * s)) + (f2 == (A)0 ? (A)0 : f2 * (t2 + d2 * s2));
  s = (m == ninf ? s : f1 * s) + (m2 == ninf ? s2 : f2 * s2);
  m = mn;
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const LogprobArgs a) {
  using S = LpAcc<T>;
  using A = typename S::type;
  const A ninf = -(A)__builtin_huge_valf();
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.M) return;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  A m = ninf, s = (A)0, t = (A)0;
  for (int64_t v = lane; v < a.V; v += 64) {
    const A z = S::load(x[v]);
    if (z == ninf) continue;
    if (z != z) {
      s = z;
      continue;
    }
    join_part<S, A>(m, s, t, z, (A)1, (A)0);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const A m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), t2 = __shfl_xor(t, o, 64);
    join_part<S, A>(m, s, t, m2, s2, t2);
  }
  const A logs = m == ninf ? (A)__builtin_nanf("") : S::log(s);
  if (lane == 0) {
    const int64_t id = a.ids[row];
    static_cast<A*>(a.logprob)[row] = id < 0 || id >= a.V ? (A)__builtin_nanf("") : S::load(x[id]) - m - logs;
    if (a.entropy != nullptr) static_cast<A*>(a.entropy)[row] = logs - t / s;
  }
  // one alternative after the other: the first in (value descending, id ascending, NaN
  // last) order behind the one before it
  A pv = (A)0;
  int64_t pi = -1;
  for (int j = 0; j < a.top; ++j) {
    A bv = (A)0;
    int64_t bi = a.V;
    auto before = [](A v1, int64_t i1, A v2, int64_t i2) {
      if (v1 != v1) return v2 != v2 && i1 < i2;
      return v2 != v2 || v1 > v2 || (v1 == v2 && i1 < i2);
    };
    for (int64_t v = lane; v < a.V; v += 64) {
      const A z = S::load(x[v]);
      if (pi >= 0 && !before(pv, pi, z, v)) continue;
      if (bi == a.V || before(z, v, bv, bi)) {
        bv = z;
        bi = v;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const A v2 = __shfl_xor(bv, o, 64);
      const int64_t i2 = __shfl_xor((long long)bi, o, 64);
      if (i2 < a.V && (bi == a.V || before(v2, i2, bv, bi))) {
        bv = v2;
        bi = i2;
      }
    }
    pv = bv;
    pi = bi;
    if (lane == 0) {
      a.top_ids[row * a.top + j] = bi;
      static_cast<A*>(a.top_logprob)[row * a.top + j] = bv - m - logs;
    }
  }
}

}  // namespace dg

using namespace dg;

extern "C" int dg_token_logprobs(int64_t M, int64_t V, int dtype, const void* x, int64_t x_ld, const int64_t* ids,
                                 void* logprob, void* entropy, int top, void* top_logprob, int64_t* top_ids,
                                 void* stream) {
  DG_REQUIRE(M >= 0 && V >= 1, DG_EINVAL, "token_logprobs: %lld rows of %lld logits", (long long)M, (long long)V);
  DG_REQUIRE(dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64, DG_EUNSUPPORTED,
             "token_logprobs: dtype %d unsupported", dtype);
  DG_REQUIRE(top >= 0 && top <= 64 && top <= V, DG_EINVAL, "token_logprobs: top %d outside [0, min(V, 64)]", top);
  DG_REQUIRE(V <= 0x7fffffff && (M + 3) / 4 <= 0x7fffffff, DG_EINVAL, "token_logprobs: too many logits or rows");
  if (M == 0) return DG_OK;
  DG_REQUIRE(x && ids && logprob && (top == 0 || (top_logprob && top_ids)), DG_EINVAL, "token_logprobs: NULL argument");
  LogprobArgs a{x, x_ld, M, V, ids, logprob, entropy, top, top_logprob, top_ids};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((M + 3) / 4));
  if (dtype == DG_F64) hipLaunchKernelGGL(token_logprobs_kernel<double>, grid, dim3(256), 0, s, a);
  else if (dtype == DG_F32) hipLaunchKernelGGL(token_logprobs_kernel<float>, grid, dim3(256), 0, s, a);
  else if (dtype == DG_BF16) hipLaunchKernelGGL(token_logprobs_kernel<bf16_t>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(token_logprobs_kernel<f16_t>, grid, dim3(256), 0, s, a);
  return check_launch("token_logprobs_kernel");
}
