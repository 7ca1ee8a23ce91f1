// Row operators over a vocabulary: log probabilities of given tokens with entropy and best alternatives, distillation
// from a teacher's best logits, and the gradient of both.
//
// Everything is computed in binary logarithms: with c = log2(e) / temperature, s_j = c * x_j and the row's largest
// logit m, S = sum_j 2^(s_j - c m), so log2 p_j = (s_j - c m) - log2 S.  A row keeps (m, log2 S).
#include "thx_rows.h"

#include "kernels/thx_common.h"

namespace thx {
namespace {

template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

constexpr double kLog2E = 1.44269504088896340735992468100189214;
constexpr double kLn2 = 0.693147180559945309417232121458176568;

THX_DEV float acc_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
THX_DEV double acc_exp2(double v) { return exp2(v); }
THX_DEV float acc_log2(float v) { return log2f(v); }
THX_DEV double acc_log2(double v) { return log2(v); }

// c * (x - m).  Half precision: one fused multiply-add against the rounded product c * m, which is the same number
// wherever the row is read, so that its rounding changes no probability; the products of single precision can overflow
// (a mask of the type's lowest value), their difference is taken first.
THX_DEV float scaled(thx_f16 x, float m, float c) { return __builtin_fmaf((float)x, c, -(m * c)); }
THX_DEV float scaled(float x, float m, float c) { return (x - m) * c; }
THX_DEV double scaled(double x, double m, double c) { return (x - m) * c; }

// log p in natural units.  In single and double precision not by way of the binary logarithm, whose factor of 1.44 would
// carry a mask of the type's lowest value beyond the type's range.
THX_DEV float log_prob(thx_f16 x, float m, float c, float, float ls) { return (scaled(x, m, c) - ls) * (float)kLn2; }
THX_DEV float log_prob(float x, float m, float, float inv_t, float ls) { return (x - m) * inv_t - ls * (float)kLn2; }
THX_DEV double log_prob(double x, double m, double, double inv_t, double ls) { return (x - m) * inv_t - ls * kLn2; }

template <class A> THX_DEV A neg_inf() { return -(A)INFINITY; }

// One value per row or per (row, entry) whose type is not worth a kernel of its own.
THX_DEV int64_t load_index(const void* p, int is64, int64_t i) { return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int*)p)[i]; }
template <class A>
THX_DEV A load_real(const void* p, int dtype, int64_t i) {
  return dtype == THX_F16 ? (A)((const thx_f16*)p)[i] : dtype == THX_F32 ? (A)((const float*)p)[i] : (A)((const double*)p)[i];
}

// The order of the alternatives as one integer: larger logits are larger numbers, NaN the largest, both zeros equal; of
// equal logits the lower column.
typedef unsigned __int128 Wide;
template <class T> struct Order {
  typedef unsigned long long Key;
  THX_DEV static Key key(T v, int64_t col) {
    const float f = (float)v + 0.0f;
    unsigned b = __float_as_uint(f);
    b = f != f ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((Key)b << 32) | (unsigned)(0xffffffffu - (unsigned)col);
  }
};
template <> struct Order<double> {
  typedef Wide Key;
  THX_DEV static Key key(double v, int64_t col) {
    const double f = v + 0.0;
    unsigned long long b = (unsigned long long)__double_as_longlong(f);
    b = f != f ? ~0ull : (b >> 63) ? ~b : b | (1ull << 63);
    return ((Key)b << 32) | (unsigned)(0xffffffffu - (unsigned)col);
  }
};
template <class Key> THX_DEV int64_t key_column(Key k) { return (int64_t)(0xffffffffu - (unsigned)k); }

template <class A, class F>
THX_DEV A block_fold(A v, A* lds, F f) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = f(v, (A)__shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  A r = lds[0];
  for (unsigned w = 1; w < blockDim.x / 64; ++w) r = f(r, lds[w]);
  return r;
}
struct Plus { template <class A> THX_DEV A operator()(A a, A b) const { return a + b; } };
struct Most { template <class A> THX_DEV A operator()(A a, A b) const { return a > b ? a : b; } };

// Largest logit and sums of a row; every thread of the block gets them.
template <class A> struct Sums { A m, s, w; };  // max, sum 2^d, sum d 2^d with d = scaled(x, m)

template <class T, class A>
THX_DEV Sums<A> row_sums(const T* x, int64_t cols, A c, A* lds) {
  A m = neg_inf<A>();
  for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) m = Most()(m, (A)x[j]);
  m = block_fold(m, lds, Most());
  const A ref = m == neg_inf<A>() ? (A)0 : m;
  A s = 0, w = 0;
  for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
    const A d = scaled(x[j], ref, c), e = acc_exp2(d);
    s += e;
    w += e * (d < (A)-30000 ? (A)-30000 : d);
  }
  Sums<A> r;
  r.m = m;
  r.s = block_fold(s, lds, Plus());
  r.w = block_fold(w, lds, Plus());
  return r;
}

// A row of nothing but -infinity (a NaN makes the sum a NaN).
template <class A> THX_DEV bool nothing_left(A m, A s) { return m == neg_inf<A>() && s == (A)0; }

template <class A> struct LpOut { A *log_prob, *entropy, *top; int64_t* top_at; A* stats; };

template <class T>
__global__ void __launch_bounds__(256) lp_forward(const T* x, int64_t xs, int64_t rows, int64_t cols, const void* tokens,
                                                  int64_t ts, int t64, typename AccOf<T>::type c,
                                                  typename AccOf<T>::type inv_t, int n_top, LpOut<typename AccOf<T>::type> o) {
  typedef typename AccOf<T>::type A;
  typedef typename Order<T>::Key Key;
  __shared__ A lds[4];
  __shared__ Key best[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const Sums<A> q = row_sums<T, A>(xr, cols, c, lds);
    const bool none = nothing_left(q.m, q.s);
    const A ls = none ? neg_inf<A>() : acc_log2(q.s);
    if (threadIdx.x == 0) {
      const int64_t t = load_index(tokens, t64, r * ts);
      A lp = 0;
      if (t >= cols) lp = (A)NAN;
      else if (t >= 0) lp = none ? neg_inf<A>() : log_prob(xr[t], q.m, c, inv_t, ls);
      o.log_prob[r] = lp;
      o.entropy[r] = none ? (A)0 : (ls - q.w / q.s) * (A)kLn2;
      o.stats[2 * r] = q.m;
      o.stats[2 * r + 1] = ls;
    }
    Key last = ~(Key)0;  // no column has this key: a column of 0 would need 2^32 - 1 less it
    bool first = true;
    for (int k = 0; k < n_top; ++k) {
      Key b = 0;
      for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
        const Key v = Order<T>::key(xr[j], j);
        if ((first || v < last) && v > b) b = v;
      }
      for (int m = 32; m >= 1; m >>= 1) {
        Key other;
        unsigned* w = (unsigned*)&other;
        const unsigned* mine = (const unsigned*)&b;
        for (int i = 0; i < (int)(sizeof(Key) / 4); ++i) w[i] = (unsigned)__shfl_xor((int)mine[i], m, 64);
        if (other > b) b = other;
      }
      __syncthreads();
      if ((threadIdx.x & 63) == 0) best[threadIdx.x / 64] = b;
      __syncthreads();
      for (int w = 0; w < 4; ++w)
        if (best[w] > b) b = best[w];
      last = b;
      first = false;
      if (threadIdx.x == 0) {
        const int64_t j = key_column(b);
        o.top_at[r * n_top + k] = j;
        o.top[r * n_top + k] = none ? neg_inf<A>() : log_prob(xr[j], q.m, c, inv_t, ls);
      }
    }
    __syncthreads();
  }
}

// Teacher's side of one row: largest logit and sum over the entries there are; every thread gets them.
template <class A>
THX_DEV void teacher_sums(const void* teacher, int tdt, const void* ids, int i64, int64_t t0, int64_t i0, int n, A c, A* lds,
                          A& m, A& s) {
  m = neg_inf<A>();
  for (int k = threadIdx.x; k < n; k += blockDim.x)
    if (load_index(ids, i64, i0 + k) >= 0) m = Most()(m, load_real<A>(teacher, tdt, t0 + k));
  m = block_fold(m, lds, Most());
  s = 0;
  for (int k = threadIdx.x; k < n; k += blockDim.x)
    if (load_index(ids, i64, i0 + k) >= 0)
      s += acc_exp2((load_real<A>(teacher, tdt, t0 + k) - (m == neg_inf<A>() ? (A)0 : m)) * c);
  s = block_fold(s, lds, Plus());
}

template <class A> struct Teacher { const void* logits; int64_t ls; int dtype; const void* ids; int64_t is; int i64, n; };

template <class T>
__global__ void __launch_bounds__(256) kd_forward(const T* x, int64_t xs, int64_t rows, int64_t cols,
                                                  Teacher<typename AccOf<T>::type> t, typename AccOf<T>::type c,
                                                  typename AccOf<T>::type inv_t, typename AccOf<T>::type t2,
                                                  typename AccOf<T>::type* loss,
                                                  typename AccOf<T>::type* stats) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const Sums<A> q = row_sums<T, A>(xr, cols, c, lds);
    const bool none = nothing_left(q.m, q.s);
    const A ls = none ? neg_inf<A>() : acc_log2(q.s);
    A tm, ts;
    teacher_sums<A>(t.logits, t.dtype, t.ids, t.i64, r * t.ls, r * t.is, t.n, c, lds, tm, ts);
    const bool tnone = nothing_left(tm, ts);
    const A tls = tnone ? neg_inf<A>() : acc_log2(ts);
    A sum = 0;
    for (int k = threadIdx.x; k < t.n; k += blockDim.x) {
      const int64_t id = load_index(t.ids, t.i64, r * t.is + k);
      if (id < 0) continue;
      if (id >= cols) sum = (A)NAN;
      if (id >= cols || tnone) continue;
      const A tv = load_real<A>(t.logits, t.dtype, r * t.ls + k), p = acc_exp2((tv - tm) * c - tls);
      const A lp = none ? neg_inf<A>() : log_prob(xr[id], q.m, c, inv_t, ls);
      if (!(p == (A)0)) sum += p * (log_prob(tv, tm, c, inv_t, tls) - lp);
    }
    sum = block_fold(sum, lds, Plus());
    if (q.s != q.s) sum = q.s;
    if (threadIdx.x == 0) {
      loss[r] = sum * t2;
      stats[4 * r] = q.m;
      stats[4 * r + 1] = ls;
      stats[4 * r + 2] = tm;
      stats[4 * r + 3] = tls;
    }
    __syncthreads();
  }
}

// dx_j = p_j (a + b log2 p_j) + sum_k c_k [j = id_k]: the gradient of every function of the log probabilities above.
template <class T, class A>
THX_DEV void grad_row(const T* xr, T* dr, int64_t cols, A m, A ls, A c, A a, A b) {
  const bool none = m == neg_inf<A>() && ls == neg_inf<A>();
  for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
    const A l = scaled(xr[j], none ? (A)0 : m, c) - ls, p = acc_exp2(l);
    A v = p * a;
    if (b != (A)0) v += p * b * (l < (A)-30000 ? (A)-30000 : l);
    dr[j] = none ? (T)0 : (T)v;
  }
}

template <class A>
struct LpGrad {
  const void* tokens; int64_t ts; int t64;
  const A* stats; int64_t ss;
  const A* entropy; int64_t es;
  const int64_t* top; int64_t ps; int n_top;
  const A* g; int64_t gs;
  const A* u; int64_t us;
  const A* gt; int64_t gts;
};

template <class T>
__global__ void __launch_bounds__(256) lp_backward(const T* x, int64_t xs, int64_t rows, int64_t cols,
                                                   LpGrad<typename AccOf<T>::type> q, typename AccOf<T>::type c,
                                                   typename AccOf<T>::type inv_t, T* dx) {
  typedef typename AccOf<T>::type A;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    T* dr = dx + r * cols;
    const A m = q.stats[r * q.ss], ls = q.stats[r * q.ss + 1];
    const bool none = m == neg_inf<A>() && ls == neg_inf<A>();
    int64_t t = load_index(q.tokens, q.t64, r * q.ts);
    A w = q.g && t >= 0 ? q.g[r * q.gs] : (A)0;
    A a = t >= cols && q.g ? (A)NAN : w;
    if (t >= cols) t = -1;
    for (int k = 0; k < q.n_top; ++k) a += q.gt[r * q.gts + k];
    const A u = q.u ? q.u[r * q.us] : (A)0;
    if (q.u) a += u * q.entropy[r * q.es];
    grad_row<T, A>(xr, dr, cols, m, ls, c, -a * inv_t, -u * (A)kLn2 * inv_t);
    __syncthreads();
    if (none) continue;
    for (int k = threadIdx.x; k <= q.n_top; k += blockDim.x) {
      const int64_t id = k == q.n_top ? (q.g ? t : -1) : q.top[r * q.ps + k];
      if (id < 0 || id >= cols) continue;
      A v = id == t ? w : (A)0;
      bool mine = true;
      for (int i = 0; i < q.n_top; ++i)
        if (q.top[r * q.ps + i] == id) {
          v += q.gt[r * q.gts + i];
          if (i < k) mine = false;
        }
      if (!mine) continue;
      const A l = scaled(xr[id], m, c) - ls, p = acc_exp2(l);
      A d = -p * a;
      if (u != (A)0) d -= p * u * (A)kLn2 * (l < (A)-30000 ? (A)-30000 : l);
      dr[id] = (T)((d + v) * inv_t);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) kd_backward(const T* x, int64_t xs, int64_t rows, int64_t cols,
                                                   Teacher<typename AccOf<T>::type> t,
                                                   const typename AccOf<T>::type* stats, int64_t ss,
                                                   const typename AccOf<T>::type* g, int64_t gs,
                                                   typename AccOf<T>::type c, typename AccOf<T>::type temperature, T* dx) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    T* dr = dx + r * cols;
    const A m = stats[r * ss], ls = stats[r * ss + 1], tm = stats[r * ss + 2], tls = stats[r * ss + 3];
    const bool none = m == neg_inf<A>() && ls == neg_inf<A>();
    const bool tnone = tm == neg_inf<A>() && tls == neg_inf<A>();
    const A gt = g[r * gs] * temperature;
    A bad = 0;
    for (int k = threadIdx.x; k < t.n; k += blockDim.x)
      if (load_index(t.ids, t.i64, r * t.is + k) >= cols) bad = (A)1;
    bad = block_fold(bad, lds, Most());
    A a = tnone ? (A)0 : gt;
    if (bad != (A)0) a = (A)NAN;
    grad_row<T, A>(xr, dr, cols, m, ls, c, a, (A)0);
    __syncthreads();
    if (!none && !tnone && bad == (A)0) {
      for (int k = threadIdx.x; k < t.n; k += blockDim.x) {
        const int64_t id = load_index(t.ids, t.i64, r * t.is + k);
        if (id < 0) continue;
        A v = 0;
        bool mine = true;
        for (int i = 0; i < t.n; ++i)
          if (load_index(t.ids, t.i64, r * t.is + i) == id) {
            if (i < k) mine = false;
            v += acc_exp2((load_real<A>(t.logits, t.dtype, r * t.ls + i) - tm) * c - tls);
          }
        if (mine) dr[id] = (T)(gt * (acc_exp2(scaled(xr[id], m, c) - ls) - v));
      }
    }
    __syncthreads();
  }
}

int acc_code(int dtype) { return dtype == THX_F64 ? THX_F64 : THX_F32; }
bool is_float(int dtype) { return dtype == THX_F16 || dtype == THX_F32 || dtype == THX_F64; }
unsigned grid_of(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(n, 1 << 20)); }

template <class F>
int by_type(int x, F&& f) {
  if (x == THX_F16) return f(thx_f16());
  if (x == THX_F32) return f(thx_f32());
  return f(thx_f64());
}

// The logits of a call: checked for type, width and temperature.
int logits_of(const char* what, const thx_array* x, double temperature, int flags, Rows* r) {
  int rc = rows_of(what, "logits", x, -1, 1, flags, r);
  if (rc) return rc;
  if (!is_float(r->dtype)) return fail(THX_ERR_TYPE, "%s: logits of dtype code %d", what, r->dtype);
  if (!(temperature >= 1e-6 && temperature <= 1e6))
    return fail(THX_ERR_ARG, "%s: temperature must lie between 1e-6 and 1e6", what);
  if (r->rows && !r->cols) return fail(THX_ERR_ARG, "%s: the logits have no columns", what);
  if (r->cols >= (int64_t(1) << 31)) return fail(THX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 columns", what);
  return THX_OK;
}

// One index per row, or per (row, entry): int32 or int64.
int indices_of(const char* what, const char* name, const thx_array* a, const thx_array* x, int64_t cols, int flags, Rows* r) {
  if (!a) return fail(THX_ERR_ARG, "%s: %s is missing", what, name);
  const int dt = a->dtype & ~THX_REUSED;
  if (dt != THX_I32 && dt != THX_I64) return fail(THX_ERR_TYPE, "%s: %s must be int32 or int64", what, name);
  return like_rows(what, name, a, x, dt, cols, flags, r);
}

int token_logprob(const thx_array* logits, const thx_array* tokens, double temperature, int n_top, const thx_array* log_prob,
                  const thx_array* entropy, const thx_array* top, const thx_array* top_at, const thx_array* stats, int flags) {
  const char* what = "token log probabilities";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[2], out[5];
  int rc = logits_of(what, logits, temperature, flags, &in[0]);
  if (rc) return rc;
  const int acc = acc_code(in[0].dtype);
  if (n_top < 0 || n_top > THX_MAX_TOP || (in[0].rows && n_top > in[0].cols))
    return fail(THX_ERR_ARG, "%s: %d alternatives of %lld columns (at most %d)", what, n_top, (long long)in[0].cols, THX_MAX_TOP);
  if ((rc = indices_of(what, "tokens", tokens, logits, -1, flags, &in[1]))) return rc;
  if ((rc = like_rows(what, "log_prob", log_prob, logits, acc, -1, flags, &out[0]))) return rc;
  if ((rc = like_rows(what, "entropy", entropy, logits, acc, -1, flags, &out[1]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 2, flags, &out[2]))) return rc;
  if (n_top) {
    if ((rc = like_rows(what, "top_log_probs", top, logits, acc, n_top, flags, &out[3]))) return rc;
    if ((rc = like_rows(what, "top_tokens", top_at, logits, THX_I64, n_top, flags, &out[4]))) return rc;
  }
  for (int k = 0; k < 5; ++k)
    if ((rc = contiguous_rows(what, "a result", out[k]))) return rc;
  if ((rc = no_overlap(what, out, 5, in, 2)) && !dry) return rc;
  const std::string plan = "lp|rows";
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename AccOf<T>::type A;
    A c = (A)(kLog2E / temperature), inv_t = (A)(1.0 / temperature);
    int t64 = in[1].dtype == THX_I64;
    LpOut<A> o = {(A*)out[0].ptr, (A*)out[1].ptr, (A*)out[3].ptr, (int64_t*)out[4].ptr, (A*)out[2].ptr};
    void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &in[1].ptr, &in[1].stride, &t64, &c, &inv_t, &n_top, &o};
    return launch_builtin((const void*)&lp_forward<T>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
  });
}

int token_logprob_grad(const thx_array* logits, const thx_array* tokens, const thx_array* stats, const thx_array* entropy,
                       const thx_array* top_at, const thx_array* g, const thx_array* u, const thx_array* gt,
                       double temperature, const thx_array* dx, int flags) {
  const char* what = "token log probabilities' gradient";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[8], out;
  int rc = logits_of(what, logits, temperature, flags, &in[0]);
  if (rc) return rc;
  const int acc = acc_code(in[0].dtype);
  int64_t n_top = 0;
  if (gt) {
    if (!top_at || gt->nd < 1 || gt->nd > THX_MAX_ND) return fail(THX_ERR_ARG, "%s: alternatives' gradients without their columns", what);
    n_top = gt->shape[gt->nd - 1];
    if (n_top < 1 || n_top > THX_MAX_TOP) return fail(THX_ERR_ARG, "%s: %lld alternatives", what, (long long)n_top);
    if ((rc = like_rows(what, "g_top", gt, logits, acc, n_top, flags, &in[7]))) return rc;
    if ((rc = like_rows(what, "top_tokens", top_at, logits, THX_I64, n_top, flags, &in[4]))) return rc;
  }
  if ((rc = indices_of(what, "tokens", tokens, logits, -1, flags, &in[1]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 2, flags, &in[2]))) return rc;
  if ((rc = like_rows(what, "entropy", entropy, logits, acc, -1, flags, &in[3]))) return rc;
  if (g && (rc = like_rows(what, "g_log_prob", g, logits, acc, -1, flags, &in[5]))) return rc;
  if (u && (rc = like_rows(what, "g_entropy", u, logits, acc, -1, flags, &in[6]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, in[0].dtype, in[0].cols, flags, &out))) return rc;
  if ((rc = contiguous_rows(what, "dlogits", out))) return rc;
  if ((rc = no_overlap(what, &out, 1, in, 8)) && !dry) return rc;
  const std::string plan = "lpg|rows";
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename AccOf<T>::type A;
    A c = (A)(kLog2E / temperature), inv_t = (A)(1.0 / temperature);
    LpGrad<A> q = {in[1].ptr, in[1].stride, in[1].dtype == THX_I64, (const A*)in[2].ptr, in[2].stride, (const A*)in[3].ptr,
                   in[3].stride, (const int64_t*)in[4].ptr, in[4].stride, (int)n_top, (const A*)in[5].ptr, in[5].stride,
                   (const A*)in[6].ptr, in[6].stride, (const A*)in[7].ptr, in[7].stride};
    void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &q, &c, &inv_t, &out.ptr};
    return launch_builtin((const void*)&lp_backward<T>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
  });
}

// The teacher's entries: [rows..., n] logits of any floating-point type and indices.
int teacher_of(const char* what, const thx_array* teacher, const thx_array* tokens, const thx_array* logits, int flags,
               Rows* t, Rows* ids) {
  if (!teacher || !tokens) return fail(THX_ERR_ARG, "%s: the teacher's logits or tokens are missing", what);
  const int dt = teacher->dtype & ~THX_REUSED;
  if (!is_float(dt)) return fail(THX_ERR_TYPE, "%s: teacher's logits of dtype code %d", what, dt);
  if (teacher->nd < 1 || teacher->nd > THX_MAX_ND) return fail(THX_ERR_TYPE, "%s: teacher's logits of rank %d", what, teacher->nd);
  const int64_t n = teacher->shape[teacher->nd - 1];
  if (n < 1 || n > THX_MAX_TEACHER)
    return fail(THX_ERR_ARG, "%s: %lld teacher's entries per row (1 to %d)", what, (long long)n, THX_MAX_TEACHER);
  int rc = like_rows(what, "teacher_logits", teacher, logits, dt, n, flags, t);
  if (rc) return rc;
  return indices_of(what, "teacher_tokens", tokens, logits, n, flags, ids);
}

template <class A>
Teacher<A> teacher_args(const Rows& t, const Rows& ids) {
  return {t.ptr, t.stride, t.dtype, ids.ptr, ids.stride, ids.dtype == THX_I64, (int)t.cols};
}

int topk_distill(const thx_array* logits, const thx_array* teacher, const thx_array* tokens, double temperature,
                 const thx_array* loss, const thx_array* stats, int flags) {
  const char* what = "distillation loss";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[3], out[2];
  int rc = logits_of(what, logits, temperature, flags, &in[0]);
  if (rc) return rc;
  const int acc = acc_code(in[0].dtype);
  if ((rc = teacher_of(what, teacher, tokens, logits, flags, &in[1], &in[2]))) return rc;
  if ((rc = like_rows(what, "loss", loss, logits, acc, -1, flags, &out[0]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 4, flags, &out[1]))) return rc;
  for (int k = 0; k < 2; ++k)
    if ((rc = contiguous_rows(what, "a result", out[k]))) return rc;
  if ((rc = no_overlap(what, out, 2, in, 3)) && !dry) return rc;
  const std::string plan = "kd|rows";
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename AccOf<T>::type A;
    A c = (A)(kLog2E / temperature), inv_t = (A)(1.0 / temperature), t2 = (A)(temperature * temperature);
    Teacher<A> q = teacher_args<A>(in[1], in[2]);
    void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &q, &c, &inv_t, &t2, &out[0].ptr, &out[1].ptr};
    return launch_builtin((const void*)&kd_forward<T>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
  });
}

int topk_distill_grad(const thx_array* logits, const thx_array* teacher, const thx_array* tokens, const thx_array* stats,
                      const thx_array* g, double temperature, const thx_array* dx, int flags) {
  const char* what = "distillation loss's gradient";
  const bool dry = (flags & THX_DRY_RUN) != 0;
  Rows in[5], out;
  int rc = logits_of(what, logits, temperature, flags, &in[0]);
  if (rc) return rc;
  const int acc = acc_code(in[0].dtype);
  if ((rc = teacher_of(what, teacher, tokens, logits, flags, &in[1], &in[2]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 4, flags, &in[3]))) return rc;
  if ((rc = like_rows(what, "g_loss", g, logits, acc, -1, flags, &in[4]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, in[0].dtype, in[0].cols, flags, &out))) return rc;
  if ((rc = contiguous_rows(what, "dlogits", out))) return rc;
  if ((rc = no_overlap(what, &out, 1, in, 5)) && !dry) return rc;
  const std::string plan = "kdg|rows";
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename AccOf<T>::type A;
    A c = (A)(kLog2E / temperature), tt = (A)temperature;
    Teacher<A> q = teacher_args<A>(in[1], in[2]);
    void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &q, &in[3].ptr, &in[3].stride, &in[4].ptr,
                    &in[4].stride, &c, &tt, &out.ptr};
    return launch_builtin((const void*)&kd_backward<T>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
  });
}

}  // namespace
}  // namespace thx

using namespace thx;

extern "C" {

int thx_token_logprob_workspace(const thx_array* logits, int n_top, size_t* nbytes) {
  return guarded("thx_token_logprob_workspace", [&] {
    if (!logits || !nbytes) return fail(THX_ERR_ARG, "thx_token_logprob_workspace: null argument");
    *nbytes = 0;
    return (int)THX_OK;
  });
}

int thx_token_logprob_call(const thx_array* logits, const thx_array* tokens, double temperature, int n_top,
                           const thx_array* log_prob, const thx_array* entropy, const thx_array* top_log_probs,
                           const thx_array* top_tokens, const thx_array* stats, void* workspace,
                           size_t workspace_bytes, int flags) {
  return guarded("thx_token_logprob_call", [&] {
    return token_logprob(logits, tokens, temperature, n_top, log_prob, entropy, top_log_probs, top_tokens, stats, flags);
  });
}

int thx_token_logprob_grad_call(const thx_array* logits, const thx_array* tokens, const thx_array* stats,
                                const thx_array* entropy, const thx_array* top_tokens, const thx_array* g_log_prob,
                                const thx_array* g_entropy, const thx_array* g_top, double temperature,
                                const thx_array* dlogits, int flags) {
  return guarded("thx_token_logprob_grad_call", [&] {
    return token_logprob_grad(logits, tokens, stats, entropy, top_tokens, g_log_prob, g_entropy, g_top, temperature, dlogits,
                              flags);
  });
}

int thx_topk_distill_workspace(const thx_array* logits, size_t* nbytes) {
  return guarded("thx_topk_distill_workspace", [&] {
    if (!logits || !nbytes) return fail(THX_ERR_ARG, "thx_topk_distill_workspace: null argument");
    *nbytes = 0;
    return (int)THX_OK;
  });
}

int thx_topk_distill_call(const thx_array* logits, const thx_array* teacher, const thx_array* tokens, double temperature,
                          const thx_array* loss, const thx_array* stats, void* workspace, size_t workspace_bytes,
                          int flags) {
  return guarded("thx_topk_distill_call",
                 [&] { return topk_distill(logits, teacher, tokens, temperature, loss, stats, flags); });
}

int thx_topk_distill_grad_call(const thx_array* logits, const thx_array* teacher, const thx_array* tokens,
                               const thx_array* stats, const thx_array* g_loss, double temperature,
                               const thx_array* dlogits, int flags) {
  return guarded("thx_topk_distill_grad_call",
                 [&] { return topk_distill_grad(logits, teacher, tokens, stats, g_loss, temperature, dlogits, flags); });
}

}  // extern "C"
