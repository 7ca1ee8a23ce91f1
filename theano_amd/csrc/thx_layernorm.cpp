// Layer normalisation over rows and its gradients: planner and kernels.
#include "thx_rows.h"
#include "thx_rows_device.h"

namespace thx {
namespace {

// ---- rows held in registers ----------------------------------------------------------------------------------------
//
// TPR threads share a row, each holding VPT vectors of 16 bytes of it from the one time it is read: the mean, the squares
// around the mean and the result come out of registers.  Up to 64 threads of one wave need nothing but shuffles; larger
// groups are whole blocks and pass the sums of their waves through LDS.

template <int TPR> struct Block { enum { threads = TPR > 256 ? TPR : 256, rows = threads / TPR }; };

// Sums of N values over the TPR threads of a row, in every one of them.  `lds`: N values of every wave, two sets of
// them used in turn, so that one barrier a call is enough: a set is written again two calls later, and by then every
// wave has passed the barrier of the call between, behind its reads.
template <int TPR, int N, class A>
THX_DEV void row_sums(A (&v)[N], A* lds, int& turn) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    A* set = lds + (turn * Block<TPR>::rows + threadIdx.x / TPR) * N * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) set[k * W + threadIdx.x % TPR / 64] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = set[k * W];
#pragma unroll
      for (int w = 1; w < W; ++w) v[k] += set[k * W + w];
    }
  }
}

// Vector i of an array of `cols` elements; what lies behind the end is 0.
template <class T, int V>
THX_DEV void load_edge(Vec<T, V>& v, const T* p, int64_t i, int64_t cols) {
  if ((i + 1) * V <= cols) {
    load_vec<T, V, false, true>(v, p + i * V);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v.v[e] = i * V + e < cols ? p[i * V + e] : (T)0;
  }
}
template <class T, int V>
THX_DEV void store_edge(T* p, const Vec<T, V>& v, int64_t i, int64_t cols, bool nt) {
  if ((i + 1) * V <= cols) {
    store_out(p + i * V, v, nt);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i * V + e < cols) p[i * V + e] = v.v[e];
  }
}

// A thread's V sums of columns, `left` of which are there.
template <class P, class A, int V>
THX_DEV void store_sums(P* p, const A (&v)[V], int64_t left) {
  constexpr int W = Width<P>::value < V ? Width<P>::value : V;
  if (left >= V) {
#pragma unroll
    for (int e = 0; e < V; e += W) {
      Vec<P, W> o;
#pragma unroll
      for (int k = 0; k < W; ++k) o.v[k] = (P)v[e + k];
      store_out(p + e, o, false);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = (P)v[e];
  }
}

THX_DEV float rsqrt_of(float v) { return 1.0f / sqrtf(v); }
THX_DEV double rsqrt_of(double v) { return 1.0 / sqrt(v); }

// A thread with at most 16 columns keeps their parameters in registers over all the rows its block goes through, and
// loads the next row's vectors before it works on this one's.  Read anew for each row, single-precision parameters are
// twice the traffic of a half-precision row (16384 rows of 4096 halves: 60 us, and 53 with this).
template <class T, int VPT> struct Keep { enum { value = Width<T>::value * VPT <= 16 }; };

template <class T, class P, int TPR, int VPT>
__global__ void __launch_bounds__(Block<TPR>::threads) ln_forward(const T* x, int64_t xs, int64_t rows, int64_t cols,
                                                                  const P* gamma, const P* beta, double eps, T* y,
                                                                  typename AccOf<T>::type* mean,
                                                                  typename AccOf<T>::type* invstd, bool nt) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value, RPB = Block<TPR>::rows;
  constexpr bool KEEP = Keep<T, VPT>::value;
  __shared__ A lds[TPR > 64 ? 2 * Block<TPR>::threads / 64 : 1];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const A share = (A)1 / (A)cols;
  int turn = 0;
  // threads without a row repeat the last one
  auto row_at = [&](int64_t r0) { return r0 + group < rows ? r0 + group : rows - 1; };
  Vec<T, V> v[VPT], next[KEEP ? VPT : 1];
  Vec<P, V> g[KEEP ? VPT : 1], b[KEEP ? VPT : 1];
  if constexpr (KEEP) {
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      load_edge(next[u], x + row_at((int64_t)blockIdx.x * RPB) * xs, u * TPR + t, cols);
      if (gamma) load_edge(g[u], gamma, u * TPR + t, cols);
      if (beta) load_edge(b[u], beta, u * TPR + t, cols);
    }
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t r = row_at(r0);
    const int64_t rn = row_at(r0 + (int64_t)gridDim.x * RPB);
    const bool more = r0 + (int64_t)gridDim.x * RPB < rows;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      if constexpr (KEEP) {
        v[u] = next[u];
        if (more) load_edge(next[u], x + rn * xs, u * TPR + t, cols);
      } else {
        load_edge(v[u], x + r * xs, u * TPR + t, cols);
      }
    }
    A sum[1] = {0};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += (A)v[u].v[e];
    row_sums<TPR>(sum, lds, turn);
    const A mu = sum[0] * share;
    A sq[1] = {0};
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int64_t left = cols - (int64_t)(u * TPR + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A d = (A)v[u].v[e] - mu;
        sq[0] += e < left ? d * d : (A)0;
      }
    }
    row_sums<TPR>(sq, lds, turn);
    const A inv = rsqrt_of(sq[0] * share + (A)eps);
    T* yr = y + r * cols;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int64_t i = u * TPR + t;
      const int w = KEEP ? u : 0;
      if (i * V >= cols) continue;
      if constexpr (!KEEP) {
        if (gamma) load_edge(g[0], gamma, i, cols);
        if (beta) load_edge(b[0], beta, i, cols);
      }
      Vec<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        A z = ((A)v[u].v[e] - mu) * inv;
        if (gamma) z *= (A)g[w].v[e];
        if (beta) z += (A)b[w].v[e];
        o.v[e] = (T)z;
      }
      store_edge(yr, o, i, cols, nt);
    }
    if (t == 0) mean[r] = mu, invstd[r] = inv;
  }
}

// A block's sums of the parameters' gradients: the gradients themselves where it is the only one.
template <int TPR, int VPT, class P, class A, int V>
THX_DEV void leave_sums(A (&dg)[VPT][V], A (&db)[VPT][V], int group, int t, int64_t cols, A* partial, P* dgamma, P* dbeta) {
  constexpr int RPB = Block<TPR>::rows;
  // the groups of a block first, through LDS, one column vector at a time
  constexpr int VEC = V * 2;
  __shared__ A fold[RPB > 1 ? RPB * TPR * VEC : 1];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        fold[(2 * e) * RPB * TPR + threadIdx.x] = dg[u][e];
        fold[(2 * e + 1) * RPB * TPR + threadIdx.x] = db[u][e];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          for (int k = 1; k < RPB; ++k) {
            dg[u][e] += fold[(2 * e) * RPB * TPR + k * TPR + t];
            db[u][e] += fold[(2 * e + 1) * RPB * TPR + k * TPR + t];
          }
      }
    }
    if (group == 0) {
      const int64_t j = (int64_t)(u * TPR + t) * V;
      if (gridDim.x == 1) {  // nothing to join
        store_sums(dgamma + j, dg[u], cols - j);
        if (dbeta) store_sums(dbeta + j, db[u], cols - j);
      } else {
        A* to = partial + (int64_t)blockIdx.x * 2 * cols + j;
        store_sums(to, dg[u], cols - j);
        store_sums(to + cols, db[u], cols - j);
      }
    }
  }
}

// The gradients.  A block goes through rows blockIdx.x, + gridDim.x, ... (RPB of them at a time) and keeps the sums of
// dy * xhat and dy of its rows in registers, per column; at the end it leaves them in partial[block][2][cols], which
// ln_join adds up.  One pass over x and dy serves all three gradients.
template <class T, class P, int TPR, int VPT, bool PARAMS>
__global__ void __launch_bounds__(Block<TPR>::threads) ln_backward(const T* x, int64_t xs, const T* dy, int64_t ds,
                                                                   int64_t rows, int64_t cols, const P* gamma,
                                                                   const typename AccOf<T>::type* mean, int64_t ms,
                                                                   const typename AccOf<T>::type* invstd, int64_t is, T* dx,
                                                                   typename AccOf<T>::type* partial, P* dgamma, P* dbeta,
                                                                   bool nt) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value, RPB = Block<TPR>::rows;
  __shared__ A lds[TPR > 64 ? 4 * Block<TPR>::threads / 64 : 1];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const A share = (A)1 / (A)cols;
  int turn = 0;
  A dg[PARAMS ? VPT : 1][V], db[PARAMS ? VPT : 1][V];
#pragma unroll
  for (int u = 0; u < (PARAMS ? VPT : 1); ++u)
#pragma unroll
    for (int e = 0; e < V; ++e) dg[u][e] = db[u][e] = 0;
  // the next row's vectors are on their way while this one's are worked on, where registers are left for them
  constexpr bool AHEAD = TPR < 1024 || V * VPT < 16;
  auto row_at = [&](int64_t r0) { return r0 + group < rows ? r0 + group : rows - 1; };
  Vec<T, V> v[VPT], d[VPT], vn[VPT], dn[VPT];
  Vec<P, V> g[VPT];
  A mn = 0, in = 0;
  auto load = [&](int64_t r) {
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      load_edge(vn[u], x + r * xs, u * TPR + t, cols);
      load_edge(dn[u], dy + r * ds, u * TPR + t, cols);  // 0 behind the end: those columns add nothing
    }
    mn = mean[r * ms];
    in = invstd[r * is];
  };
  if (AHEAD && (int64_t)blockIdx.x * RPB < rows) load(row_at((int64_t)blockIdx.x * RPB));
#pragma unroll
  for (int u = 0; u < VPT; ++u)
    if (gamma) load_edge(g[u], gamma, u * TPR + t, cols);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const bool live = r0 + group < rows;
    const int64_t r = row_at(r0);
    if (!AHEAD) load(r);
    const A mu = mn, inv = in;
#pragma unroll
    for (int u = 0; u < VPT; ++u) v[u] = vn[u], d[u] = dn[u];
    if (AHEAD && r0 + (int64_t)gridDim.x * RPB < rows) load(row_at(r0 + (int64_t)gridDim.x * RPB));
    A s[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A dv = (A)d[u].v[e], a = gamma ? dv * (A)g[u].v[e] : dv, xh = ((A)v[u].v[e] - mu) * inv;
        s[0] += a;
        s[1] += a * xh;
        if (PARAMS && live) {
          dg[u][e] += dv * xh;
          db[u][e] += dv;
        }
      }
    }
    row_sums<TPR>(s, lds, turn);
    s[0] *= share;
    s[1] *= share;
    T* out = dx + r * cols;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int64_t i = u * TPR + t;
      if (i * V >= cols) continue;
      Vec<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A dv = (A)d[u].v[e], a = gamma ? dv * (A)g[u].v[e] : dv, xh = ((A)v[u].v[e] - mu) * inv;
        o.v[e] = (T)(inv * (a - s[0] - xh * s[1]));
      }
      store_edge(out, o, i, cols, nt);
    }
  }
  if constexpr (PARAMS) leave_sums<TPR, VPT>(dg, db, group, t, cols, partial, dgamma, dbeta);
}

// Forward and all gradients in one, for a dy that is known beforehand: a row and its dy are read once.  The sums behind
// dx need no invstd until they are there, sum(a xhat) = invstd sum(a (x - mean)), so that the row's sums come together in
// two steps: the mean, then the squares around it beside both others.
template <class T, class P, int TPR, int VPT, bool PARAMS>
__global__ void __launch_bounds__(Block<TPR>::threads) ln_train(const T* x, int64_t xs, const T* dy, int64_t ds, int64_t rows,
                                                                int64_t cols, const P* gamma, const P* beta, double eps, T* y,
                                                                typename AccOf<T>::type* mean,
                                                                typename AccOf<T>::type* invstd, T* dx,
                                                                typename AccOf<T>::type* partial, P* dgamma, P* dbeta, bool nt) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value, RPB = Block<TPR>::rows, WAVES = Block<TPR>::threads / 64;
  __shared__ A lds_mean[TPR > 64 ? 2 * WAVES : 1], lds[TPR > 64 ? 6 * WAVES : 1];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const A share = (A)1 / (A)cols;
  int turn_mean = 0, turn = 0;
  A dg[VPT][V], db[VPT][V];
#pragma unroll
  for (int u = 0; u < VPT; ++u)
#pragma unroll
    for (int e = 0; e < V; ++e) dg[u][e] = db[u][e] = 0;
  constexpr bool AHEAD = TPR < 1024 || V * VPT < 16;
  auto row_at = [&](int64_t r0) { return r0 + group < rows ? r0 + group : rows - 1; };
  Vec<T, V> v[VPT], d[VPT], vn[VPT], dn[VPT];
  Vec<P, V> g[VPT];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      load_edge(vn[u], x + r * xs, u * TPR + t, cols);
      load_edge(dn[u], dy + r * ds, u * TPR + t, cols);
    }
  };
  if (AHEAD && (int64_t)blockIdx.x * RPB < rows) load(row_at((int64_t)blockIdx.x * RPB));
#pragma unroll
  for (int u = 0; u < VPT; ++u)
    if (gamma) load_edge(g[u], gamma, u * TPR + t, cols);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const bool live = r0 + group < rows;
    const int64_t r = row_at(r0);
    if (!AHEAD) load(r);
#pragma unroll
    for (int u = 0; u < VPT; ++u) v[u] = vn[u], d[u] = dn[u];
    if (AHEAD && r0 + (int64_t)gridDim.x * RPB < rows) load(row_at(r0 + (int64_t)gridDim.x * RPB));
    A sum[1] = {0};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += (A)v[u].v[e];
    row_sums<TPR>(sum, lds_mean, turn_mean);
    const A mu = sum[0] * share;
    A s[3] = {0, 0, 0};
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int64_t left = cols - (int64_t)(u * TPR + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A dv = (A)d[u].v[e], a = gamma ? dv * (A)g[u].v[e] : dv, xc = (A)v[u].v[e] - mu;
        s[0] += e < left ? xc * xc : (A)0;
        s[1] += a;
        s[2] += a * xc;
      }
    }
    row_sums<TPR>(s, lds, turn);
    const A inv = rsqrt_of(s[0] * share + (A)eps), s0 = s[1] * share, s1 = s[2] * share * inv;
    T *yr = y + r * cols, *out = dx + r * cols;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int64_t i = u * TPR + t;
      if (i * V >= cols) continue;
      Vec<P, V> b;
      if (beta) load_edge(b, beta, i, cols);
      Vec<T, V> o, z;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A dv = (A)d[u].v[e], gv = gamma ? (A)g[u].v[e] : (A)1, xh = ((A)v[u].v[e] - mu) * inv;
        const A w = gamma ? xh * gv : xh;
        z.v[e] = (T)(beta ? w + (A)b.v[e] : w);
        o.v[e] = (T)(inv * ((gamma ? dv * gv : dv) - s0 - xh * s1));
        if (PARAMS && live) {
          dg[u][e] += dv * xh;
          db[u][e] += dv;
        }
      }
      store_edge(yr, z, i, cols, nt);
      store_edge(out, o, i, cols, nt);
    }
    if (t == 0) mean[r] = mu, invstd[r] = inv;
  }
  if constexpr (PARAMS) leave_sums<TPR, VPT>(dg, db, group, t, cols, partial, dgamma, dbeta);
}

// Adds up the blocks' sums: 64 columns by 16 slices of the blocks to a block here, blockIdx.y 0 for gamma, 1 for beta.
template <class A, class P>
__global__ void __launch_bounds__(1024) ln_join(const A* partial, int blocks, int64_t cols, P* dgamma, P* dbeta) {
  __shared__ A lds[16][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x / 64;
  P* to = blockIdx.y ? dbeta : dgamma;
  const A* from = partial + (blockIdx.y ? cols : 0);
  for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < cols; c0 += (int64_t)gridDim.x * 64) {
    const int64_t c = c0 + lane;
    A s = 0;
    if (c < cols) {
      int k = slice;
      for (; k + 48 < blocks; k += 64) {
        const A p0 = from[(int64_t)k * 2 * cols + c], p1 = from[(int64_t)(k + 16) * 2 * cols + c];
        const A p2 = from[(int64_t)(k + 32) * 2 * cols + c], p3 = from[(int64_t)(k + 48) * 2 * cols + c];
        s += (p0 + p1) + (p2 + p3);
      }
      for (; k < blocks; k += 16) s += from[(int64_t)k * 2 * cols + c];
    }
    lds[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && c < cols) {
#pragma unroll
      for (int k = 1; k < 16; ++k) s += lds[k][lane];
      to[c] = (P)s;
    }
    __syncthreads();
  }
}

// ---- any row -------------------------------------------------------------------------------------------------------
//
// Rows beyond what a block of 1024 threads holds, and parameters that do not lie side by side: one block per row, read
// once per step (the later reads come from the caches), and the parameters' sums by columns in a pass of their own.

template <class A>
THX_DEV A block_sum(A v, A* lds) {
  v = lanes_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  A r = lds[0];
  for (unsigned w = 1; w < blockDim.x / 64; ++w) r += lds[w];
  return r;
}

template <class T, class P>
__global__ void __launch_bounds__(1024) ln_forward_any(const T* x, int64_t xs, int64_t rows, int64_t cols, const P* gamma, int64_t gs,
                                                  const P* beta, int64_t bs, double eps, T* y,
                                                  typename AccOf<T>::type* mean, typename AccOf<T>::type* invstd) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[16];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    A s = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) s += (A)xr[c];
    const A mu = block_sum(s, lds) / (A)cols;
    s = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const A d = (A)xr[c] - mu;
      s += d * d;
    }
    const A inv = (A)1 / (A)sqrt(block_sum(s, lds) / (A)cols + (A)eps);
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      A v = ((A)xr[c] - mu) * inv;
      if (gamma) v *= (A)gamma[c * gs];
      if (beta) v += (A)beta[c * bs];
      y[r * cols + c] = (T)v;
    }
    if (threadIdx.x == 0) mean[r] = mu, invstd[r] = inv;
  }
}

template <class T, class P>
__global__ void __launch_bounds__(1024) ln_backward_any(const T* x, int64_t xs, const T* dy, int64_t ds, int64_t rows, int64_t cols,
                                                    const P* gamma, int64_t gs, const typename AccOf<T>::type* mean,
                                                    int64_t ms, const typename AccOf<T>::type* invstd, int64_t is, T* dx) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[16];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * xs, *dr = dy + r * ds;
    const A mu = mean[r * ms], inv = invstd[r * is];
    A s1 = 0, s2 = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const A a = gamma ? (A)dr[c] * (A)gamma[c * gs] : (A)dr[c];
      s1 += a;
      s2 += a * (((A)xr[c] - mu) * inv);
    }
    s1 = block_sum(s1, lds) / (A)cols;
    s2 = block_sum(s2, lds) / (A)cols;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const A a = gamma ? (A)dr[c] * (A)gamma[c * gs] : (A)dr[c];
      dx[r * cols + c] = (T)(inv * (a - s1 - ((A)xr[c] - mu) * inv * s2));
    }
  }
}

// Sums over a slice of the rows, one column per thread: partial[slice][2][cols].
template <class T>
__global__ void __launch_bounds__(1024) ln_params_any(const T* x, int64_t xs, const T* dy, int64_t ds, int64_t rows,
                                                      int64_t cols, const typename AccOf<T>::type* mean, int64_t ms,
                                                      const typename AccOf<T>::type* invstd, int64_t is,
                                                      typename AccOf<T>::type* partial) {
  typedef typename AccOf<T>::type A;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = (int64_t)blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < cols; c += (int64_t)gridDim.x * blockDim.x) {
    A g = 0, b = 0;
    for (int64_t r = r0; r < r1; ++r) {
      const A d = (A)dy[r * ds + c];
      g += d * (((A)x[r * xs + c] - mean[r * ms]) * invstd[r * is]);
      b += d;
    }
    partial[(int64_t)blockIdx.y * 2 * cols + c] = g;
    partial[((int64_t)blockIdx.y * 2 + 1) * cols + c] = b;
  }
}

int acc_code(int dtype) { return dtype == THX_F64 ? THX_F64 : THX_F32; }

int check_types(const char* what, int x, int p) {
  if (x != THX_F16 && x != THX_F32 && x != THX_F64) return fail(THX_ERR_TYPE, "%s: rows of dtype code %d", what, x);
  if (p >= 0 && p != x && !(x == THX_F16 && p == THX_F32))
    return fail(THX_ERR_TYPE, "%s: parameters of dtype code %d beside rows of %d", what, p, x);
  return THX_OK;
}

// A parameter: one value per column, at any stride (0 repeats one value).
int param_of(const char* what, const char* name, const thx_array* a, int dtype, int64_t cols, int flags, Rows* r) {
  int rc = rows_of(what, name, a, dtype, 0, flags, r);
  if (rc) return rc;
  if (a->nd != 1 || a->shape[0] != cols)
    return fail(THX_ERR_SHAPE, "Input dimension mis-match. (%s: %s does not have one value for each of %lld columns)", what,
                name, (long long)cols);
  return THX_OK;
}

unsigned grid_of(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(n, 1 << 20)); }

// How a call's rows are laid out over threads; tpr 0: the kernels for any row.
struct Shape {
  int tpr = 0, vpt = 0;
};

// The smallest group of threads that holds a row in registers; tpr 0 where none does or a parameter's values do not lie
// side by side.  Forward 16 columns to a thread, with their parameters kept: rows of 4096 halves as 256 threads x 2
// vectors 53 us, 64 x 8 87 us (parameters read for every row), rows of 1024 floats 64 x 4 48 us, 256 x 1 53 us.  Backward
// a thread keeps two sums more per column: rows of 1024 floats 128 x 2 78 us, 64 x 4 81 us, of 8192 halves 1024 x 1 87 us,
// 512 x 2 101 us.
Shape shape_of(int64_t cols, int dtype, bool backward, bool packed) {
  static const Shape halves[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {128, 2}, {256, 2}, {512, 2}, {1024, 2}, {1024, 4}, {1024, 8}};
  static const Shape words[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {128, 4}, {256, 4}, {512, 4}, {1024, 4}, {1024, 8}};
  static const Shape back[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {128, 2}, {256, 2}, {1024, 1}, {1024, 2}};
  const int isz = dtype_size(dtype);
  const int64_t vectors = (cols * isz + 15) / 16;
  auto first = [&](const Shape* s, int n) {
    for (int k = 0; k < n; ++k)
      if (vectors <= (int64_t)s[k].tpr * s[k].vpt) return s[k];
    return Shape();
  };
  if (!packed || !cols) return Shape();
  return backward ? first(back, 9) : isz == 2 ? first(halves, 11) : first(words, 11);
}

// Blocks for rows in groups of as many as a block takes at once: at most `most`, each with the same number of turns.
int64_t even_blocks(const Shape& s, int64_t rows, int64_t most) {
  const int64_t per = s.tpr > 256 ? 1 : 256 / s.tpr, groups = (rows + per - 1) / per;
  const int64_t turns = std::max<int64_t>(1, (groups + most - 1) / most);
  return std::max<int64_t>(1, (groups + turns - 1) / turns);
}

// As many threads as the device holds.
int64_t forward_blocks(const Shape& s, int64_t rows) {
  return even_blocks(s, rows, (int64_t)compute_units() * (2048 / std::max(256, s.tpr)));
}

// Every block leaves one set of sums for ln_join, so no more of them than it takes to keep the memory busy: rows of 4096
// halves, 256 x 2, with 2, 3 and 4 blocks to a compute unit 82, 85 and 89 us, and ln_join 8 to 11.
// What one block does in four turns it does alone, and writes the gradients itself: 4 rows of 4096 halves 9.2 us, where
// four blocks take 6.1 and ln_join 6.2; 8 rows in one block 14 us.
int64_t backward_blocks(const Shape& s, int64_t rows) {
  if (rows <= 4 * (s.tpr > 256 ? 1 : 256 / s.tpr)) return 1;
  return even_blocks(s, rows, (int64_t)compute_units() * (s.tpr > 256 ? 1 : s.vpt > 1 ? 2 : 4));
}

int slices_of(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(64, rows / 64)); }

// f(integral constants TPR, VPT) for a shape.
template <int TPR, int VPT> struct Held { enum { tpr = TPR, vpt = VPT }; };
template <class F>
int by_shape_halves(const Shape& s, F&& f) {
  switch (s.tpr * 16 + s.vpt) {
    case 8 * 16 + 1: return f(Held<8, 1>());
    case 16 * 16 + 1: return f(Held<16, 1>());
    case 32 * 16 + 1: return f(Held<32, 1>());
    case 64 * 16 + 1: return f(Held<64, 1>());
    case 64 * 16 + 2: return f(Held<64, 2>());
    case 128 * 16 + 2: return f(Held<128, 2>());
    case 256 * 16 + 2: return f(Held<256, 2>());
    case 512 * 16 + 2: return f(Held<512, 2>());
    case 1024 * 16 + 2: return f(Held<1024, 2>());
    case 1024 * 16 + 4: return f(Held<1024, 4>());
    default: return f(Held<1024, 8>());
  }
}
template <class F>
int by_shape_words(const Shape& s, F&& f) {
  switch (s.tpr * 16 + s.vpt) {
    case 8 * 16 + 1: return f(Held<8, 1>());
    case 16 * 16 + 1: return f(Held<16, 1>());
    case 32 * 16 + 1: return f(Held<32, 1>());
    case 64 * 16 + 1: return f(Held<64, 1>());
    case 64 * 16 + 2: return f(Held<64, 2>());
    case 64 * 16 + 4: return f(Held<64, 4>());
    case 128 * 16 + 4: return f(Held<128, 4>());
    case 256 * 16 + 4: return f(Held<256, 4>());
    case 512 * 16 + 4: return f(Held<512, 4>());
    case 1024 * 16 + 4: return f(Held<1024, 4>());
    default: return f(Held<1024, 8>());
  }
}
template <class T, class F>
int by_shape(const Shape& s, F&& f) {
  if constexpr (sizeof(T) == 2) return by_shape_halves(s, f);
  else return by_shape_words(s, f);
}
template <class F>
int by_back_shape(const Shape& s, F&& f) {
  switch (s.tpr * 16 + s.vpt) {
    case 8 * 16 + 1: return f(Held<8, 1>());
    case 16 * 16 + 1: return f(Held<16, 1>());
    case 32 * 16 + 1: return f(Held<32, 1>());
    case 64 * 16 + 1: return f(Held<64, 1>());
    case 64 * 16 + 2: return f(Held<64, 2>());
    case 128 * 16 + 2: return f(Held<128, 2>());
    case 256 * 16 + 2: return f(Held<256, 2>());
    case 1024 * 16 + 1: return f(Held<1024, 1>());
    default: return f(Held<1024, 2>());
  }
}

std::string plan_of(const char* name, int dtype, const Shape& s) {
  return std::string(name) + "|t" + std::to_string(dtype) +
         (s.tpr ? "|r" + std::to_string(s.tpr) + "x" + std::to_string(s.vpt) : std::string("|any"));
}

// f(T(), P()) for the element types of the rows and of the parameters.
template <class F>
int by_types(int x, int p, F&& f) {
  if (x == THX_F16) return p == THX_F32 ? f(thx_f16(), thx_f32()) : f(thx_f16(), thx_f16());
  if (x == THX_F32) return f(thx_f32(), thx_f32());
  return f(thx_f64(), thx_f64());
}

int layernorm(const thx_array* x, const thx_array* gamma, const thx_array* beta, double epsilon, const thx_array* y,
              const thx_array* mean, const thx_array* invstd, int flags) {
  const char* what = "layer normalization";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[3], out[3];
  int rc = rows_of(what, "x", x, -1, 1, flags, &in[0]);
  if (rc) return rc;
  if (beta && !gamma) return fail(THX_ERR_ARG, "%s: beta without gamma", what);
  if (!(epsilon >= 0)) return fail(THX_ERR_ARG, "%s: epsilon must be at least 0", what);
  const int pt = gamma ? gamma->dtype & ~THX_REUSED : in[0].dtype;
  if ((rc = check_types(what, in[0].dtype, pt))) return rc;
  if (gamma && (rc = param_of(what, "gamma", gamma, pt, in[0].cols, flags, &in[1]))) return rc;
  if (beta && (rc = param_of(what, "beta", beta, pt, in[0].cols, flags, &in[2]))) return rc;
  if ((rc = like_rows(what, "y", y, x, in[0].dtype, in[0].cols, flags, &out[0]))) return rc;
  if ((rc = like_rows(what, "mean", mean, x, acc_code(in[0].dtype), -1, flags, &out[1]))) return rc;
  if ((rc = like_rows(what, "invstd", invstd, x, acc_code(in[0].dtype), -1, flags, &out[2]))) return rc;
  for (int k = 0; k < 3; ++k)
    if ((rc = contiguous_rows(what, "a result", out[k]))) return rc;
  if ((rc = no_overlap(what, out, 3, in, 3)) && !dry) return rc;
  const bool packed = (!gamma || in[0].cols <= 1 || in[1].stride == 1) && (!beta || in[0].cols <= 1 || in[2].stride == 1);
  const Shape shape = shape_of(in[0].cols, in[0].dtype, false, packed);
  const std::string plan = plan_of("ln", in[0].dtype, shape);
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  bool nt = stream_out(in[0], out[0]);
  return by_types(in[0].dtype, pt, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    if (!shape.tpr) {
      void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &in[1].ptr, &in[1].stride, &in[2].ptr,
                      &in[2].stride, &epsilon, &out[0].ptr, &out[1].ptr, &out[2].ptr};
      return launch_builtin((const void*)&ln_forward_any<T, P>, plan, dim3(grid_of(in[0].rows)), dim3(1024), args);
    }
    return by_shape<T>(shape, [&](auto h) {
      constexpr int TPR = decltype(h)::tpr, VPT = decltype(h)::vpt;
      void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &in[1].ptr, &in[2].ptr, &epsilon, &out[0].ptr,
                      &out[1].ptr, &out[2].ptr, &nt};
      return launch_builtin((const void*)&ln_forward<T, P, TPR, VPT>, plan,
                            dim3(grid_of(forward_blocks(shape, in[0].rows))), dim3(Block<TPR>::threads), args);
    });
  });
}

// Blocks that leave sums of the parameters' gradients, for either family of kernels.
int64_t partial_blocks(const Rows& x, bool packed) {
  const Shape s = shape_of(x.cols, x.dtype, true, packed);
  return s.tpr ? backward_blocks(s, x.rows) : slices_of(x.rows);
}

int layernorm_grad_bytes(const thx_array* x, const thx_array* dgamma, size_t* nbytes) {
  if (!x || !nbytes) return fail(THX_ERR_ARG, "layer normalization gradient: null argument");
  Rows r;
  int rc = rows_of("layer normalization gradient", "x", x, -1, 1, THX_DRY_RUN, &r);
  if (rc) return rc;
  // whichever gamma's stride asks for
  const int64_t blocks = std::max(partial_blocks(r, true), partial_blocks(r, false));
  *nbytes = dgamma ? (size_t)blocks * 2 * r.cols * dtype_size(acc_code(r.dtype)) : 0;
  return THX_OK;
}

int layernorm_grad(const thx_array* x, const thx_array* dy, const thx_array* gamma, const thx_array* mean,
                   const thx_array* invstd, const thx_array* dx, const thx_array* dgamma, const thx_array* dbeta,
                   void* ws, size_t ws_bytes, int flags) {
  const char* what = "layer normalization gradient";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[5], out[3];
  int rc = rows_of(what, "x", x, -1, 1, flags, &in[0]);
  if (rc) return rc;
  const int acc = acc_code(in[0].dtype);
  if ((dgamma || dbeta) && !gamma) return fail(THX_ERR_ARG, "%s: gradients of parameters without gamma", what);
  if (dbeta && !dgamma) return fail(THX_ERR_ARG, "%s: dbeta without dgamma", what);
  const int pt = gamma ? gamma->dtype & ~THX_REUSED : in[0].dtype;
  if ((rc = check_types(what, in[0].dtype, pt))) return rc;
  if ((rc = like_rows(what, "dy", dy, x, in[0].dtype, in[0].cols, flags, &in[1]))) return rc;
  if ((rc = like_rows(what, "mean", mean, x, acc, -1, flags, &in[2]))) return rc;
  if ((rc = like_rows(what, "invstd", invstd, x, acc, -1, flags, &in[3]))) return rc;
  if (gamma && (rc = param_of(what, "gamma", gamma, pt, in[0].cols, flags, &in[4]))) return rc;
  if ((rc = like_rows(what, "dx", dx, x, in[0].dtype, in[0].cols, flags, &out[0]))) return rc;
  if (dgamma && (rc = param_of(what, "dgamma", dgamma, pt, in[0].cols, flags, &out[1]))) return rc;
  if (dbeta && (rc = param_of(what, "dbeta", dbeta, pt, in[0].cols, flags, &out[2]))) return rc;
  for (int k = 0; k < 3; ++k)
    if ((rc = contiguous_rows(what, "a result", out[k]))) return rc;
  if ((rc = no_overlap(what, out, 3, in, 5)) && !dry) return rc;
  size_t need = 0;
  if ((rc = layernorm_grad_bytes(x, dgamma, &need))) return rc;
  if ((rc = check_workspace(what, ws, ws_bytes, need, flags))) return rc;
  const bool packed = !gamma || in[0].cols <= 1 || in[4].stride == 1;
  const Shape shape = shape_of(in[0].cols, in[0].dtype, true, packed);
  const std::string plan = plan_of("lng", in[0].dtype, shape);
  set_last_plan(plan);
  if (dry || !in[0].cols) return THX_OK;
  if ((rc = ensure_init())) return rc;
  bool nt = stream_out(in[0], out[0]);
  return by_types(in[0].dtype, pt, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    typedef typename AccOf<T>::type A;
    int rc = THX_OK;
    int blocks = (int)partial_blocks(in[0], packed);
    const unsigned columns = grid_of((in[0].cols + 63) / 64);
    if (shape.tpr) {
      rc = by_back_shape(shape, [&](auto h) {
        constexpr int TPR = decltype(h)::tpr, VPT = decltype(h)::vpt;
        void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[4].ptr,
                        &in[2].ptr, &in[2].stride, &in[3].ptr, &in[3].stride, &out[0].ptr, &ws, &out[1].ptr, &out[2].ptr,
                        &nt};
        const void* kernel = dgamma ? (const void*)&ln_backward<T, P, TPR, VPT, true>
                                    : (const void*)&ln_backward<T, P, TPR, VPT, false>;
        return launch_builtin(kernel, plan, dim3(blocks), dim3(Block<TPR>::threads), args);
      });
    } else {
      if (in[0].rows) {
        void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[4].ptr,
                        &in[4].stride, &in[2].ptr, &in[2].stride, &in[3].ptr, &in[3].stride, &out[0].ptr};
        rc = launch_builtin((const void*)&ln_backward_any<T, P>, plan, dim3(grid_of(in[0].rows)), dim3(1024), args);
      }
      if (!rc && dgamma) {
        void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[2].ptr,
                        &in[2].stride, &in[3].ptr, &in[3].stride, &ws};
        rc = launch_builtin((const void*)&ln_params_any<T>, plan, dim3(grid_of((in[0].cols + 255) / 256), blocks), dim3(256),
                            args);
      }
    }
    if (rc || !dgamma || (shape.tpr && blocks == 1)) return rc;
    void* join[] = {&ws, &blocks, &in[0].cols, &out[1].ptr, &out[2].ptr};
    return launch_builtin((const void*)&ln_join<A, P>, plan + "|join", dim3(columns, dbeta ? 2 : 1), dim3(1024), join);
  });
}

int layernorm_train(const thx_array* x, const thx_array* dy, const thx_array* gamma, const thx_array* beta, double epsilon,
                    const thx_array* y, const thx_array* mean, const thx_array* invstd, const thx_array* dx,
                    const thx_array* dgamma, const thx_array* dbeta, void* ws, size_t ws_bytes, int flags) {
  const char* what = "layer normalization with gradients";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  // what the two calls look at, then what lies between them
  int rc = layernorm(x, gamma, beta, epsilon, y, mean, invstd, flags | THX_DRY_RUN);
  if (rc) return rc;
  if ((rc = layernorm_grad(x, dy, gamma, mean, invstd, dx, dgamma, dbeta, ws, ws_bytes, flags | THX_DRY_RUN))) return rc;
  Rows in[4], out[6];
  const thx_array* ins[4] = {x, dy, gamma, beta};
  const thx_array* outs[6] = {y, mean, invstd, dx, dgamma, dbeta};
  for (int k = 0; k < 4; ++k)
    if (ins[k] && (rc = rows_of(what, "an operand", ins[k], -1, k < 2, flags, &in[k]))) return rc;
  for (int k = 0; k < 6; ++k)
    if (outs[k] && (rc = rows_of(what, "a result", outs[k], -1, k == 0 || k == 3, flags, &out[k]))) return rc;
  if ((rc = no_overlap(what, out, 6, in, 4)) && !dry) return rc;
  size_t need = 0;
  if ((rc = layernorm_grad_bytes(x, dgamma, &need))) return rc;
  if ((rc = check_workspace(what, ws, ws_bytes, need, flags))) return rc;
  const int64_t cols = in[0].cols;
  const bool packed = cols <= 1 || ((!gamma || in[2].stride == 1) && (!beta || in[3].stride == 1));
  const Shape shape = shape_of(cols, in[0].dtype, true, packed);
  // Two launches for rows that no block holds, and where a block of 1024 has no registers left for both passes and many
  // rows to go through: 2048 rows of 16384 halves 83 us, in one launch 92 (of 8192 halves 70 and 64, of 8192 floats 130
  // and 113, 16384 rows of 4096 halves 137 and 126).
  const bool crowded = in[0].dtype == THX_F16 && shape.tpr == 1024 && shape.vpt == 2 && dgamma && in[0].rows > compute_units();
  if (!shape.tpr || crowded) {
    if ((rc = layernorm(x, gamma, beta, epsilon, y, mean, invstd, flags))) return rc;
    return layernorm_grad(x, dy, gamma, mean, invstd, dx, dgamma, dbeta, ws, ws_bytes, flags);
  }
  const std::string plan = plan_of("lnt", in[0].dtype, shape);
  set_last_plan(plan);
  if (dry) return THX_OK;
  if ((rc = ensure_init())) return rc;
  bool nt = stream_out(in[0], out[3]);
  return by_types(in[0].dtype, gamma ? in[2].dtype : in[0].dtype, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    typedef typename AccOf<T>::type A;
    int blocks = (int)backward_blocks(shape, in[0].rows);
    int rc = by_back_shape(shape, [&](auto h) {
      constexpr int TPR = decltype(h)::tpr, VPT = decltype(h)::vpt;
      void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[2].ptr, &in[3].ptr,
                      &epsilon, &out[0].ptr, &out[1].ptr, &out[2].ptr, &out[3].ptr, &ws, &out[4].ptr, &out[5].ptr, &nt};
      const void* kernel = dgamma ? (const void*)&ln_train<T, P, TPR, VPT, true> : (const void*)&ln_train<T, P, TPR, VPT, false>;
      return launch_builtin(kernel, plan, dim3(blocks), dim3(Block<TPR>::threads), args);
    });
    if (rc || !dgamma || blocks == 1) return rc;
    void* join[] = {&ws, &blocks, &in[0].cols, &out[4].ptr, &out[5].ptr};
    return launch_builtin((const void*)&ln_join<A, P>, plan + "|join", dim3(grid_of((cols + 63) / 64), dbeta ? 2 : 1), dim3(1024),
                          join);
  });
}

}  // namespace
}  // namespace thx

using namespace thx;

extern "C" {

int thx_layernorm_call(const thx_array* x, const thx_array* gamma, const thx_array* beta, double epsilon,
                       const thx_array* y, const thx_array* mean, const thx_array* invstd, int flags) {
  return guarded("thx_layernorm_call", [&] { return layernorm(x, gamma, beta, epsilon, y, mean, invstd, flags); });
}

int thx_layernorm_grad_workspace(const thx_array* x, const thx_array* dgamma, size_t* nbytes) {
  return guarded("thx_layernorm_grad_workspace", [&] { return layernorm_grad_bytes(x, dgamma, nbytes); });
}

int thx_layernorm_grad_call(const thx_array* x, const thx_array* dy, const thx_array* gamma, const thx_array* mean,
                            const thx_array* invstd, const thx_array* dx, const thx_array* dgamma,
                            const thx_array* dbeta, void* workspace, size_t workspace_bytes, int flags) {
  return guarded("thx_layernorm_grad_call", [&] {
    return layernorm_grad(x, dy, gamma, mean, invstd, dx, dgamma, dbeta, workspace, workspace_bytes, flags);
  });
}

int thx_layernorm_train_call(const thx_array* x, const thx_array* dy, const thx_array* gamma, const thx_array* beta,
                             double epsilon, const thx_array* y, const thx_array* mean, const thx_array* invstd,
                             const thx_array* dx, const thx_array* dgamma, const thx_array* dbeta, void* workspace,
                             size_t workspace_bytes, int flags) {
  return guarded("thx_layernorm_train_call", [&] {
    return layernorm_train(x, dy, gamma, beta, epsilon, y, mean, invstd, dx, dgamma, dbeta, workspace, workspace_bytes, flags);
  });
}

}  // extern "C"
