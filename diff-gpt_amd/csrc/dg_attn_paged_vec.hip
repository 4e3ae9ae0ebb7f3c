// Attention over a cache in pages for a few fp32 (token, head) rows of a key head: a decode
// step.  The fp32 matrix instructions take 32 rows whatever there are; here keys and values
// go straight into registers and the products run on the vector units, bound by HBM where rows
// are few (which: paged_vec_rows).
//
// LPK = D / 8 lanes share a key (eight dims each, two 16-byte loads), a wave has KPS = 64 / LPK
// keys at a time and U times as many in flight, the four waves of a workgroup take turns.
// A group of lanes keeps a softmax state of its own for every row; the groups, then the
// waves join at the end, and splits as everywhere (seq_join4_kernel).
#include "dg_paged.h"
#include "dg_prefill.h"

namespace dg {

// D: 16, 32, 64, 128 or 256, a head of fewer dims is computed as the next; R rows, the last
// repeated where there are fewer.
template <int D, int R>
__global__ __launch_bounds__(256) void paged_vec_kernel(const SeqArgs a) {
  constexpr int LPK = D / 8, KPS = 64 / LPK, U = R <= 4 ? (KPS <= 16 ? 4 : 2) : (KPS <= 32 ? 2 : 1);
  constexpr int STEP = U * KPS;  // keys of a wave's turn, 64 at most
  static_assert(STEP <= 64, "a lane for every key's page");
  __shared__ float joined[4][R][LPK * 8 + 2];
  SeqPiece pc;
  if (!seq_piece<kPaged>(a, pc)) return;  // whole workgroups, before any barrier
  const int lane = threadIdx.x & 63, sub = lane % LPK, grp = lane / LPK;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool in = 8 * sub < a.D;  // the lane's dims are some of the head's, all eight or four of them
  const bool in2 = 8 * sub + 4 < a.D;
  const int nrows = pc.rows;
  float q[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(r, nrows - 1), qi = row / a.G;
    const float* p = static_cast<const float*>(a.q) + pc.b * a.qb + qi * a.qt + (int64_t)(pc.kvh * a.G + row - qi * a.G) * a.qh;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f}, y = x;
    if (in) x = *reinterpret_cast<const f32x4_t*>(p + 8 * sub);
    if (in2) y = *reinterpret_cast<const f32x4_t*>(p + 8 * sub + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      q[r][e] = x[e];
      q[r][4 + e] = y[e];
    }
  }
  const float* const kh = static_cast<const float*>(a.k) + (int64_t)pc.kvh * a.kh + 8 * sub;
  const float* const vh = static_cast<const float*>(a.v) + (int64_t)pc.kvh * a.vh + 8 * sub;
  const int mask = (1 << a.page_log2) - 1;
  float m[R], l[R], lc[R], o[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = kNegInf;
    l[r] = lc[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
  }

  // lane j holds the page of key j of the wave's next turn, not looked at before
  auto page_of = [&](int t0) __attribute__((always_inline)) {
    return a.table[pc.b * a.table_ld + (min(t0 + lane, pc.kend - 1) >> a.page_log2)];
  };
  int t0 = pc.kbeg + wv * STEP;
  int ids = t0 < pc.kend ? page_of(t0) : -1;
  for (; t0 < pc.kend; t0 += 4 * STEP) {
    f32x4_t kx[U], ky[U], vx[U], vy[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * KPS + grp;
      const int id = __shfl(ids, u * KPS + grp, 64);
      const bool held = id >= 0 && id < a.pages && t < pc.kend;
      const float* kp = kh + (held ? id : 0) * a.kb + (t & mask) * a.kt;
      const float* vp = vh + (held ? id : 0) * a.vb + (t & mask) * a.vt;
      kx[u] = ky[u] = vx[u] = vy[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (held && in) {
        kx[u] = *reinterpret_cast<const f32x4_t*>(kp);
        vx[u] = *reinterpret_cast<const f32x4_t*>(vp);
      }
      if (held && in2) {
        ky[u] = *reinterpret_cast<const f32x4_t*>(kp + 4);
        vy[u] = *reinterpret_cast<const f32x4_t*>(vp + 4);
      }
    }
    if (t0 + 4 * STEP < pc.kend) ids = page_of(t0 + 4 * STEP);
    // whether every row sees every key of the turn
    const bool open = t0 + STEP <= min(pc.own + 1, pc.kend);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * KPS + grp;
      float s[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_fmaf(q[r][e], kx[u][e], d);
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_fmaf(q[r][4 + e], ky[u][e], d);
        s[r] = group_sum_dpp<LPK>(d);
      }
      bool seen[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        seen[r] = open || (t < pc.kend && t <= pc.own + min(r, nrows - 1) / a.G);
        if (!seen[r]) s[r] = kNegInf;
      }
      if (a.scores != nullptr && sub == 0 && t < pc.kend) {
        float* const so = a.scores + (pc.b * a.Hkv + pc.kvh) * (int64_t)(a.N * a.G) * a.scores_ld + t;
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (r < nrows) so[r * a.scores_ld] = s[r];
      }
      bool raise = false;
#pragma unroll
      for (int r = 0; r < R; ++r) raise = raise || s[r] * a.scale_log2 > m[r] + kLazyLog2;
      if (__builtin_amdgcn_ballot_w64(raise) != 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float x = s[r] * a.scale_log2;
          const float mn = x > m[r] + kLazyLog2 ? __builtin_floorf(x) : m[r];
          const float f = m[r] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m[r] - mn);
          m[r] = mn;
          l[r] *= f;
          lc[r] *= f;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[r][e] *= f;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale_log2, m[r] == kNegInf ? 0.f : -m[r]));
        add_rounded(l[r], lc[r], p);
        if (open) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[r][e] = __builtin_fmaf(p, vx[u][e], o[r][e]);
            o[r][4 + e] = __builtin_fmaf(p, vy[u][e], o[r][4 + e]);
          }
        } else {  // a hidden key's values, NaN and infinities included, reach nothing
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[r][e] = seen[r] ? __builtin_fmaf(p, vx[u][e], o[r][e]) : o[r][e];
            o[r][4 + e] = seen[r] ? __builtin_fmaf(p, vy[u][e], o[r][4 + e]) : o[r][4 + e];
          }
        }
      }
    }
  }

  // ---- the lane groups' states joined, then the waves' ----------------------------------
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
#pragma unroll
    for (int x = LPK; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float f = m[r] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[r] - top);
    // a state without a key has zeros; a NaN is taken along
    m[r] = top;
    l[r] = sum_over_groups<LPK>((l[r] - lc[r]) * f);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = sum_over_groups<LPK>(o[r][e] * f);
  }
  if (wv > 0 && grp == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int e = 0; e < 8; ++e) joined[wv][r][8 * sub + e] = o[r][e];
      if (sub == 0) {
        joined[wv][r][8 * LPK] = m[r];
        joined[wv][r][8 * LPK + 1] = l[r];
      }
    }
  }
  __syncthreads();
  if (wv > 0 || grp > 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float m2 = joined[w][r][8 * LPK], l2 = joined[w][r][8 * LPK + 1];
      const float mn = fmaxf(m[r], m2);
      const float f1 = m[r] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[r] - mn);
      const float f2 = m2 == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
      m[r] = mn;
      l[r] = l[r] * f1 + l2 * f2;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] = o[r][e] * f1 + joined[w][r][8 * sub + e] * f2;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= nrows) break;
    const int64_t row = (pc.b * a.Hkv + pc.kvh) * (int64_t)(a.N * a.G) + r;
    if (a.nsplit > 1) {
      const int64_t part = row * a.nsplit + pc.split;
      float* wo = static_cast<float*>(a.ws_o) + part * D + 8 * sub;
      *reinterpret_cast<f32x4_t*>(wo) = f32x4_t{o[r][0], o[r][1], o[r][2], o[r][3]};
      *reinterpret_cast<f32x4_t*>(wo + 4) = f32x4_t{o[r][4], o[r][5], o[r][6], o[r][7]};
      if (sub == 0) {
        float* ml = static_cast<float*>(a.ws_ml) + 2 * part;
        ml[0] = m[r];
        ml[1] = l[r];
      }
      continue;
    }
    const int qi = r / a.G;
    const bool none = qi >= pc.count;
    if (a.lse != nullptr && sub == 0)
      static_cast<float*>(a.lse)[row] = none ? __builtin_huge_valf() : m[r] + __builtin_amdgcn_logf(l[r]);
    const float inv = 1.0f / l[r];
    float* yp = static_cast<float*>(a.y) + pc.b * a.yb + qi * a.yt + (int64_t)(pc.kvh * a.G + r - qi * a.G) * a.yh + 8 * sub;
    f32x4_t y0, y1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y0[e] = none ? 0.f : o[r][e] * inv;
      y1[e] = none ? 0.f : o[r][4 + e] * inv;
    }
    if (in) *reinterpret_cast<f32x4_t*>(yp) = y0;
    if (in2) *reinterpret_cast<f32x4_t*>(yp + 4) = y1;
  }
}

namespace {

template <int D>
int launch_vec_rows(const SeqArgs& a, dim3 grid, hipStream_t s) {
  constexpr int MOST = paged_vec_rows(D);
  const int R = a.N * a.G;
  if (R > MOST) return DG_EUNSUPPORTED;
  if (R <= 1) hipLaunchKernelGGL((paged_vec_kernel<D, 1>), grid, dim3(256), 0, s, a);
  else if (R <= 2) hipLaunchKernelGGL((paged_vec_kernel<D, 2>), grid, dim3(256), 0, s, a);
  else if constexpr (MOST >= 4) {
    if (R <= 4) hipLaunchKernelGGL((paged_vec_kernel<D, 4>), grid, dim3(256), 0, s, a);
    else if constexpr (MOST >= 8) hipLaunchKernelGGL((paged_vec_kernel<D, 8>), grid, dim3(256), 0, s, a);
  }
  return check_launch("paged_vec_kernel");
}

}  // namespace

int launch_paged_vec(const SeqArgs& a, unsigned blocks, hipStream_t s) {
  const dim3 grid(blocks);
  const int D = seq_mfma_dim(a.D);
  if (D == 16) return launch_vec_rows<16>(a, grid, s);
  if (D == 32) return launch_vec_rows<32>(a, grid, s);
  if (D == 64) return launch_vec_rows<64>(a, grid, s);
  if (D == 128) return launch_vec_rows<128>(a, grid, s);
  return launch_vec_rows<256>(a, grid, s);
}

}  // namespace dg
