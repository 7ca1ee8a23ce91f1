// Row operators over a vocabulary: log probabilities of given tokens with entropy and best alternatives, distillation
// from a teacher's best logits, and the gradient of both.
//
// Everything is computed in binary logarithms: with c = log2(e) / temperature, s_j = c * x_j and the row's largest
// logit m, S = sum_j 2^(s_j - c m), so log2 p_j = (s_j - c m) - log2 S.  A row keeps (m, log2 S).
#include <type_traits>

#include "thx_rows.h"
#include "thx_rows_device.h"

namespace thx {
namespace {

constexpr double kLog2E = 1.44269504088896340735992468100189214;
constexpr double kLn2 = 0.693147180559945309417232121458176568;

THX_DEV float acc_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
THX_DEV double acc_exp2(double v) { return exp2(v); }
THX_DEV float acc_log2(float v) { return log2f(v); }
THX_DEV double acc_log2(double v) { return log2(v); }

// The rounded product: never the first half of a fused multiply-add.
template <class A>
THX_DEV A product(A a, A b) {
#pragma clang fp contract(off)
  return a * b;
}

template <class A> THX_DEV A neg_inf() { return -(A)INFINITY; }

// The exponents c * (x - m).  FUSED, half precision at ordinary temperatures: one fused multiply-add against the product
// c * m, which is rounded, but to the same number wherever the row is read, so that it shifts all exponents of a row and
// their log2 S alike.  That product has to stay below 2^24 for any logit, which keeps the shift within half a unit; at
// temperatures under 0.0057 it need not, and the shift can pass the exponents that a float has (a largest logit of 10000
// at 1e-6: 2^368 in place of 2^0).  There, and in single and double precision, whose products can overflow as well (a mask
// of the type's lowest value), the difference is taken first.  For half precision that is two operations more to an element:
// 8192 rows of 50257 with their gradient 366 us in place of 346.
template <class T, bool FUSED = false>
struct Exponents {
  typedef typename AccOf<T>::type A;
  A c;  // log2(e) / temperature
  // What the exponents of a row are taken against, 0 while m is -infinity.
  THX_DEV A reference(A m) const { return m == neg_inf<A>() ? (A)0 : FUSED ? product(m, c) : m; }
  THX_DEV A of(A x, A ref) const { return FUSED ? __builtin_fmaf(x, c, -ref) : (x - ref) * c; }
  THX_DEV A between(A ref, A other) const { return FUSED ? ref - other : (ref - other) * c; }  // references
  // log p in natural units.  Where the difference comes first not by way of the binary logarithm, whose factor of 1.44
  // would carry a mask of the type's lowest value beyond the type's range.
  THX_DEV A log_prob(A x, A m, A inv_t, A ls) const {
    return FUSED ? (of(x, product(m, c)) - ls) * (A)kLn2 : (x - m) * inv_t - ls * (A)kLn2;
  }
};

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
  typedef unsigned Value;
  typedef unsigned long long Key;  // value, then 2^32 - 1 - column
  THX_DEV static Value value(float v) {
    const float f = v + 0.0f;
    const unsigned b = __float_as_uint(f);
    return f != f ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  }
  THX_DEV static float inverse(Value v) { return __uint_as_float((v & 0x80000000u) ? v & 0x7fffffffu : ~v); }
  THX_DEV static Value value_of(Key k) { return (Value)(k >> 32); }
  THX_DEV static Key key(T v, int64_t col) { return ((Key)value((float)v) << 32) | (unsigned)(0xffffffffu - (unsigned)col); }
  THX_DEV static Key nan_key(int64_t col) { return ((Key)0xffffffffu << 32) | (unsigned)(0xffffffffu - (unsigned)col); }
};
template <> struct Order<double> {
  typedef unsigned long long Value;
  typedef Wide Key;
  THX_DEV static Value value(double v) {
    const double f = v + 0.0;
    const unsigned long long b = (unsigned long long)__double_as_longlong(f);
    return f != f ? ~0ull : (b >> 63) ? ~b : b | (1ull << 63);
  }
  THX_DEV static double inverse(Value v) { return __longlong_as_double((long long)((v >> 63) ? v & ~(1ull << 63) : ~v)); }
  THX_DEV static Value value_of(Key k) { return (Value)(k >> 32); }
  THX_DEV static Key key(double v, int64_t col) { return ((Key)value(v) << 32) | (unsigned)(0xffffffffu - (unsigned)col); }
  THX_DEV static Key nan_key(int64_t col) { return ((Key)~0ull << 32) | (unsigned)(0xffffffffu - (unsigned)col); }
};
template <class Key> THX_DEV int64_t key_column(Key k) { return (int64_t)(0xffffffffu - (unsigned)k); }

// ---- one wave over a part of a row ----------------------------------------------------------------------------------
//
// A part of a row is read once, 64 lanes x kUnroll vectors of 16 bytes at a time.  Each lane keeps the largest logit m
// of its columns and the sums s = sum 2^d and w = sum d 2^d of the exponents d against m; they are rescaled when m grows, which
// soon happens rarely.  While m is -infinity the exponents are taken against 0: all of them are 0, or NaN, which stays.

constexpr int kUnroll = 4;
constexpr int kWaves = 4;     // waves of a block; each works alone
constexpr int kList = 512;    // candidates a wave can hold

template <class T, bool ENT, bool FUSED = false>
struct LaneSums {
  typedef typename AccOf<T>::type A;
  typedef Exponents<T, FUSED> Ex;
  A m, s, w;
  A ref;  // what the exponents are taken against
  THX_DEV void init() {
    m = neg_inf<A>();
    s = w = ref = 0;
  }
  // d 2^d is 0 where 2^d is, for d = -infinity as well
  THX_DEV static float bounded(float d) { return __builtin_fmaxf(d, -30000.0f); }
  THX_DEV static double bounded(double d) { return __builtin_fmax(d, -30000.0); }
  THX_DEV void raise(A to, const Ex& ex) {  // to > m
    const A old = ref;
    ref = ex.reference(to);
    // between the references as they were rounded, not between the logits
    const A d = m == neg_inf<A>() ? neg_inf<A>() : ex.between(old, ref), k = acc_exp2(d);
    m = to;
    if (ENT) w = k * (w + bounded(d) * s);
    s *= k;
  }
  THX_DEV void add(A x, const Ex& ex) {
    const A d = ex.of(x, ref), e = acc_exp2(d);
    s += e;
    if (ENT) w += e * bounded(d);
  }
  // Takes in the sums of other columns.
  THX_DEV void join(A om, A os, A ow, const Ex& ex) {
    LaneSums o;
    o.m = om, o.s = os, o.w = ow;
    o.ref = ex.reference(om);
    if (om > m) raise(om, ex);
    else if (m > om) o.raise(m, ex);
    s += o.s;
    if (ENT) w += o.w;
  }
  THX_DEV void join_lanes(const Ex& ex) {
    const A all = wave_largest(m);
    if (all > m) raise(all, ex);
    s = lanes_sum<64>(s);
    if (ENT) w = lanes_sum<64>(w);
  }
  // A row of nothing but -infinity (a NaN makes the sum a NaN).
  THX_DEV bool nothing_left() const { return m == neg_inf<A>() && s == (A)0; }
  THX_DEV A log2_sum() const { return nothing_left() ? neg_inf<A>() : acc_log2(s); }
};

// Largest of a vector, NaN left aside.
typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef _Float16 Half4 __attribute__((ext_vector_type(4)));
typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
THX_DEV float vector_max(const Vec<thx_f16, 8>& v) {
  const Half8 h = *(const Half8*)&v;
  const Half4 a = __builtin_elementwise_max(h.lo, h.hi);
  const Half2 b = __builtin_elementwise_max(a.lo, a.hi);
  return __builtin_fmaxf((float)b.x, (float)b.y);
}
THX_DEV float vector_max(const Vec<float, 4>& v) {
  return __builtin_fmaxf(__builtin_fmaxf(v.v[0], v.v[1]), __builtin_fmaxf(v.v[2], v.v[3]));
}
THX_DEV double vector_max(const Vec<double, 2>& v) { return __builtin_fmax(v.v[0], v.v[1]); }

THX_DEV void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
THX_DEV unsigned lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// ---- the best columns ------------------------------------------------------------------------------------------------
//
// The k best columns of a part lie in its k best vectors of 16 bytes, a vector standing for its largest value (and its
// place: of equal vectors the lower one).  Collecting vectors costs the pass one comparison of the maximum it needs
// anyway; the columns are picked out of the k vectors at the end.  `reached` is a value that k vectors are known to have:
// the k-th largest of what the 64 lanes have each seen (k <= 64), taken anew after 1, 2, 4, 8 ... steps; vectors below
// it are passed over.  What reaches it goes to a list in LDS.  Where equal values fill the list, its k best are kept
// exactly, and from then on only larger values count (equal ones lie further back in the row).
template <class T>
struct Best {
  typedef typename AccOf<T>::type A;
  typedef typename Order<T>::Key Key;
  typedef typename Order<T>::Value Value;
  Key* list;     // kList entries of this wave
  int n, k;
  A reached;     // k vectors have this much
  A limit;       // what a further vector has to have
  bool closed;   // the list holds k NaN: nothing is larger
  THX_DEV void init(Key* l, int top) {
    list = l;
    n = 0;
    k = top;
    reached = limit = neg_inf<A>();
    closed = false;
  }
  // The k-th largest of the lanes' values, bit by bit.
  THX_DEV A kth_of_lanes(A v) const {
    const Value mine = Order<T>::value(v);
    Value p = 0;
    for (int b = (int)sizeof(Value) * 8 - 1; b >= 0; --b) {
      const Value t = p | ((Value)1 << b);
      if (__popcll(__ballot(mine >= t)) >= k) p = t;
    }
    return p ? Order<T>::inverse(p) : neg_inf<A>();
  }
  THX_DEV void tighten(A lane_max) {
    const A l = kth_of_lanes(lane_max);
    if (l > reached) reached = l;
    if (l > limit) limit = l;
  }
  THX_DEV void append(bool take, Key key) {
    const unsigned long long mask = __ballot(take);
    if (take) list[n + (int)lanes_below(mask)] = key;
    n += __popcll(mask);
  }
  // Drops what k vectors are known to exceed.
  THX_DEV void sweep() {
    const Value v = Order<T>::value(reached);
    const int lane = threadIdx.x & 63, had = n;
    n = 0;
    for (int i = 0; i < had; i += 64) {
      wave_fence();
      const Key key = i + lane < had ? list[i + lane] : (Key)0;
      wave_fence();
      append(i + lane < had && Order<T>::value_of(key) >= v, key);
    }
    wave_fence();
  }
  // Puts the largest `keep` entries to the front in falling order.
  THX_DEV void sort(int keep) {
    const int lane = threadIdx.x & 63;
    Key key[kList / 64];
    int rank[kList / 64];
#pragma unroll
    for (int i = 0; i < kList / 64; ++i) {
      key[i] = i * 64 + lane < n ? list[i * 64 + lane] : (Key)0;
      rank[i] = 0;
    }
    const int used = (n + 63) / 64;
    for (int j = 0; j < n; j += 4) {  // four entries on their way at once
      Key other[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) other[a] = list[j + a < n ? j + a : n - 1];
#pragma unroll
      for (int i = 0; i < kList / 64; ++i)
        if (i < used)
#pragma unroll
          for (int a = 0; a < 4; ++a) rank[i] += j + a < n && other[a] > key[i];
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < kList / 64; ++i)
      if (i * 64 + lane < n && rank[i] < keep) list[rank[i]] = key[i];
    wave_fence();
    n = n < keep ? n : keep;
  }
  // Room for `more` entries.
  THX_DEV void make_room(int more, A lane_max) {
    if (n + more <= kList) return;
    tighten(lane_max);
    sweep();
    if (n + more <= kList) return;
    sort(k);
    const Value v = Order<T>::value_of(list[k - 1]);
    if (v == (Value)~(Value)0) closed = true;
    else limit = Order<T>::inverse(v + 1);  // the next larger value (NaN above infinity: no comparison holds)
  }
};

// The sums of the vectors [lo, hi) of a row, and its best vectors.
template <class T, bool ENT, bool TOP, bool FUSED>
THX_DEV void read_part(const T* x, int64_t cols, int64_t lo, int64_t hi, const Exponents<T, FUSED>& ex,
                       LaneSums<T, ENT, FUSED>& sum, Best<T>& best) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value;
  const int lane = threadIdx.x & 63;
  const int64_t whole = cols / V;  // vectors that are not cut off by the end of the row
  sum.init();
  int steps = 0, next = 1;
  for (int64_t at = lo; at < hi; at += 64 * kUnroll) {
    Vec<T, V> v[kUnroll];
    if (at + 64 * kUnroll <= hi && at + 64 * kUnroll <= whole) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) load_vec<T, V, false, true>(v[u], x + (at + u * 64 + lane) * V);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = at + u * 64 + lane;
        if (i < hi && i < whole) {
          load_vec<T, V, false, true>(v[u], x + i * V);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[u].v[e] = i < hi && i * V + e < cols ? x[i * V + e] : (T)neg_inf<A>();
        }
      }
    }
    A vm[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) vm[u] = vector_max(v[u]);
    A m = vm[0];
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) m = m > vm[u] ? m : vm[u];
    if (m > sum.m) sum.raise(m, ex);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int e = 0; e < V; ++e) sum.add((A)v[u].v[e], ex);
      // one vector after the other: with 32 exponentials at once the half-precision kernel takes 181 registers, not 116
      if constexpr (TOP && sizeof(T) < 8) asm volatile("" : "+v"(sum.s), "+v"(sum.w));
    }
    if constexpr (TOP) {
      if (++steps == next) {
        best.tighten(sum.m);
        next *= 2;
      }
      const bool odd = sum.s != sum.s;  // NaN (or +infinity) somewhere in this lane's columns
      if (__ballot(m >= best.limit || odd) && !best.closed) {
        best.make_room(64 * kUnroll, sum.m);
        if (!best.closed) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            const int64_t i = at + u * 64 + lane;
            bool nan = false;
            if (odd) {
#pragma unroll
              for (int e = 0; e < V; ++e) nan |= v[u].v[e] != v[u].v[e];
            }
            best.append(i < hi && (vm[u] >= best.limit || nan),
                        nan ? Order<T>::nan_key(i) : Order<T>::key((T)vm[u], i));
          }
          wave_fence();
        }
      }
    }
  }
  if constexpr (TOP) {
    if (steps * 2 != next) best.tighten(sum.m);  // not right behind the last time
    best.sweep();
    best.sort(best.k);
  }
}

// ---- results of a row, by one wave -------------------------------------------------------------------------------------

template <class A> struct LpOut { A *log_prob, *entropy, *top; int64_t* top_at; A* stats; };

template <class T>
struct LpRow {  // what lp_forward needs besides the logits
  typedef typename AccOf<T>::type A;
  const void* tokens;
  int64_t ts;
  int t64, n_top;
  A inv_t;
  LpOut<A> o;
};

// The best columns out of the best vectors (in best.list, falling), and everything else of the row; `sum` joined.
template <class T, bool TOP, bool FUSED>
THX_DEV void finish(const LpRow<T>& q, const T* x, int64_t cols, int64_t r, const Exponents<T, FUSED>& ex,
                    const LaneSums<T, true, FUSED>& sum, Best<T>& best) {
  typedef typename AccOf<T>::type A;
  typedef typename Order<T>::Key Key;
  constexpr int V = Width<T>::value;
  const int lane = threadIdx.x & 63;
  const bool none = sum.nothing_left();
  const A ls = sum.log2_sum();
  if (lane == 0) {
    const int64_t t = load_index(q.tokens, q.t64, r * q.ts);
    A lp = 0;
    if (t >= cols) lp = (A)NAN;
    else if (t >= 0) lp = none ? neg_inf<A>() : ex.log_prob((A)x[t], sum.m, q.inv_t, ls);
    q.o.log_prob[r] = lp;
    q.o.entropy[r] = none ? (A)0 : (ls - sum.w / sum.s) * (A)kLn2;
    q.o.stats[2 * r] = sum.m;
    q.o.stats[2 * r + 1] = ls;
  }
  if constexpr (TOP) {
    const int vectors = best.n, k = best.k;  // fewer vectors than k: all there are
    const Key least = vectors >= k ? best.list[k - 1] : (Key)0;
    constexpr int kMost = THX_MAX_TOP * V / 64;
    Key key[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int e = i * 64 + lane;  // element e % V of vector e / V
      key[i] = 0;
      if (e < vectors * V) {
        const int64_t j = key_column(best.list[e / V]) * V + e % V;
        if (j < cols) key[i] = Order<T>::key(x[j], j);
      }
    }
    wave_fence();
    best.n = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      best.append(key[i] != (Key)0 && Order<T>::value_of(key[i]) >= Order<T>::value_of(least), key[i]);
    wave_fence();
    best.sort(k);
    if (lane < k) {
      // there are k columns, and the list holds the k best: the look costs nothing, and no key becomes an address without it
      const int64_t j = lane < best.n ? key_column(best.list[lane]) : cols;
      const bool there = j < cols;
      q.o.top_at[r * k + lane] = there ? j : -1;
      q.o.top[r * k + lane] = !there ? (A)NAN : none ? neg_inf<A>() : ex.log_prob((A)x[j], sum.m, q.inv_t, ls);
    }
  }
}

template <class A> struct Teacher { const void* logits; int64_t ls; int dtype; const void* ids; int64_t is; int i64, n; };

template <class T>
struct KdRow {
  typedef typename AccOf<T>::type A;
  Teacher<A> t;
  A inv_t, t2;
  A *loss, *stats;
};

// An entry of the teacher: its token (-1 for none) and logit.
template <class A> struct Entry { int64_t id; A logit; };
template <class A>
THX_DEV Entry<A> load_entry(const Teacher<A>& t, int64_t r, int k) {
  return {load_index(t.ids, t.i64, r * t.is + k), load_real<A>(t.logits, t.dtype, r * t.ls + k)};
}

// An entry into the teacher's sums: nothing where it stands for no token, NaN where it names one that is not there, which
// makes the row's loss and gradient NaN.
template <class A>
THX_DEV void take_entry(const Entry<A>& e, int64_t cols, const Exponents<A>& ex, LaneSums<A, false>& ts) {
  if (e.id < 0) return;
  if (e.logit > ts.m) ts.raise(e.logit, ex);
  ts.add(e.logit, ex);
  if (e.id >= cols) ts.s = (A)NAN;
}

// q (log q - log p) of an entry, `at` being its column's logit; 0 where q is, or where it stands for no token.
template <class T, class A, bool FUSED>
THX_DEV A entry_loss(const KdRow<T>& q, const Entry<A>& e, T at, int64_t cols, const Exponents<T, FUSED>& ex,
                     const LaneSums<T, false, FUSED>& sum, A ls, A tm, A tls) {
  const Exponents<A> tex = {ex.c};
  if (e.id < 0 || (tm == neg_inf<A>() && tls == neg_inf<A>())) return 0;
  const A p = acc_exp2(tex.of(e.logit, tm) - tls);
  if (p == (A)0) return 0;
  if (e.id >= cols) return (A)NAN;
  const A lp = sum.nothing_left() ? neg_inf<A>() : ex.log_prob((A)at, sum.m, q.inv_t, ls);
  return p * (tex.log_prob(e.logit, tm, q.inv_t, tls) - lp);
}

// The logit of an entry's column, anything where it has none.
template <class T, class A>
THX_DEV T entry_at(const Entry<A>& e, const T* x, int64_t cols) {
  return e.id >= 0 && e.id < cols ? x[e.id] : (T)0;
}

template <class T, bool FUSED>
THX_DEV void finish(const KdRow<T>& q, const T* x, int64_t cols, int64_t r, const Exponents<T, FUSED>& ex,
                    const LaneSums<T, false, FUSED>& sum) {
  typedef typename AccOf<T>::type A;
  const Teacher<A>& t = q.t;
  const int lane = threadIdx.x & 63;
  const A ls = sum.log2_sum();
  LaneSums<A, false> ts;  // the teacher's side: entries as single or double precision
  const Exponents<A> tex = {ex.c};
  ts.init();
  for (int k = lane; k < t.n; k += 64) take_entry(load_entry(t, r, k), cols, tex, ts);
  ts.join_lanes(tex);
  const A tls = ts.log2_sum();
  A loss = 0;
  for (int k = lane; k < t.n; k += 64) {
    const Entry<A> e = load_entry(t, r, k);
    loss += entry_loss(q, e, entry_at(e, x, cols), cols, ex, sum, ls, ts.m, tls);
  }
  loss = lanes_sum<64>(loss);
  if (sum.s != sum.s) loss = sum.s;
  if (lane == 0) {
    q.loss[r] = loss * q.t2;
    q.stats[4 * r] = sum.m;
    q.stats[4 * r + 1] = ls;
    q.stats[4 * r + 2] = ts.m;
    q.stats[4 * r + 3] = tls;
  }
}

// ---- forward kernels ---------------------------------------------------------------------------------------------------

// The rows of a call and how they are cut: `parts` waves to a row, `per` vectors to a part.  A row of several parts leaves
// its sums in partial[row][part][3] and its best vectors (k of them, 0 for none) in lists[row][part][k].
template <class T, bool FUSED>
struct Cut {
  typedef typename AccOf<T>::type A;
  const T* x;
  int64_t xs, rows, cols;
  int64_t per;
  int parts;
  Exponents<T, FUSED> ex;
  A* partial;
  typename Order<T>::Key* lists;
};

template <class T, bool TOP, class Row, bool ENT, bool FUSED>
__global__ void __launch_bounds__(64 * kWaves) vocab_read(Cut<T, FUSED> q, Row row) {
  typedef typename Order<T>::Key Key;
  constexpr int V = Width<T>::value;
  __shared__ Key lists[TOP ? kWaves * kList : 1];
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  const int64_t units = q.rows * q.parts, vectors = (q.cols + V - 1) / V;
  for (int64_t unit = (int64_t)blockIdx.x * kWaves + wave; unit < units; unit += (int64_t)gridDim.x * kWaves) {
    const int64_t r = unit / q.parts, part = unit - r * q.parts;
    const T* x = q.x + r * q.xs;
    const int64_t lo = part * q.per, hi = lo + q.per < vectors ? lo + q.per : vectors;
    LaneSums<T, ENT, FUSED> sum;
    Best<T> best;
    int k = 0;
    if constexpr (TOP) {
      k = row.n_top;
      best.init(lists + wave * kList, k);
    }
    read_part<T, ENT, TOP>(x, q.cols, lo, hi, q.ex, sum, best);
    sum.join_lanes(q.ex);
    if (q.parts == 1) {
      if constexpr (ENT) finish<T, TOP>(row, x, q.cols, r, q.ex, sum, best);
      else finish<T>(row, x, q.cols, r, q.ex, sum);
      wave_fence();
      continue;
    }
    if (lane == 0) {
      auto* p = q.partial + unit * 3;
      p[0] = sum.m, p[1] = sum.s, p[2] = ENT ? sum.w : 0;
    }
    if (lane < k) q.lists[unit * k + lane] = lane < best.n ? best.list[lane] : (Key)0;
    wave_fence();
  }
}

// One wave per row over its parts (at most 64: one to a lane).
template <class T, bool TOP, class Row, bool ENT, bool FUSED>
__global__ void __launch_bounds__(64) vocab_join(Cut<T, FUSED> q, Row row) {
  typedef typename AccOf<T>::type A;
  typedef typename Order<T>::Key Key;
  __shared__ Key lists[TOP ? kList : 1];
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < q.rows; r += gridDim.x) {
    LaneSums<T, ENT, FUSED> sum;
    sum.init();
    if (lane < q.parts) {
      const auto* p = q.partial + (r * q.parts + lane) * 3;
      sum.join(p[0], p[1], p[2], q.ex);
    }
    sum.join_lanes(q.ex);
    const T* x = q.x + r * q.xs;
    if constexpr (ENT) {
      Best<T> best;
      if constexpr (TOP) {
        const int k = row.n_top;
        best.init(lists, k);
        // Each lane goes down the falling list of its part.  Where there are at least k parts, k entries are no less than
        // the k-th largest first entry; where the list fills up all the same, its k best are kept.
        const Key* mine = q.lists + (r * q.parts + lane) * k;
        Key at_hand[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) at_hand[i] = lane < q.parts && i < k ? mine[i] : (Key)0;
        const Key head = at_hand[0];
        best.tighten(head ? Order<T>::inverse(Order<T>::value_of(head)) : neg_inf<A>());
        const typename Order<T>::Value least = Order<T>::value(best.reached);
        Key beyond = 0;
        for (int i = 0; i < k; i += 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Key key = at_hand[j];
            at_hand[j] = lane < q.parts && i + 4 + j < k ? mine[i + 4 + j] : (Key)0;
            const bool take = key > beyond && Order<T>::value_of(key) >= least;
            if (__ballot(take) && best.n + 64 > kList) {
              wave_fence();
              best.sort(k);
              beyond = best.list[k - 1];
            }
            best.append(take && key > beyond, key);
          }
          if (!__ballot(at_hand[0] > beyond && Order<T>::value_of(at_hand[0]) >= least)) break;
        }
        wave_fence();
        best.sort(k);
        wave_fence();
      }
      finish<T, TOP>(row, x, q.cols, r, q.ex, sum, best);
    } else {
      finish<T>(row, x, q.cols, r, q.ex, sum);
    }
    wave_fence();
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------
//
// dx_j = p_j (a + b log2 p_j) + sum_k v_k [j = id_k] is the gradient of every function of the log probabilities above.
// With the exponent d of x_j against m and p_j = 2^d / S it is 2^d (a' + b' d) with a' = (a - b log2 S) / S and b' = b / S: one
// exponential and one rounding of the row's statistics per element.  The columns of the list are few; their elements are
// written once more, each by the thread of the entry that names the column first, from the sum of all entries that do.

template <class A> struct Slope { A m, ls, a, b; };

template <class A>
struct LpGrad {
  enum { kEntries = THX_MAX_TOP + 1 };
  const void* tokens; int64_t ts; int t64;
  const A* stats; int64_t ss;
  const A* entropy; int64_t es;
  const int64_t* top; int64_t ps; int n_top;
  const A* g; int64_t gs;
  const A* u; int64_t us;
  const A* gt; int64_t gts;
  A inv_t;

  THX_DEV int entries() const { return n_top + 1; }
  // The entries of row r into LDS, and the slope of the rest; called by the whole block.
  THX_DEV Slope<A> open(int64_t r, int64_t cols, int* id, A* val) const {
    const A* st = stats + r * ss;
    const int64_t t = load_index(tokens, t64, r * ts);
    const A w = g && t >= 0 ? g[r * gs] : (A)0;
    A a = t >= cols && g ? (A)NAN : w;
    for (int k = 0; k < n_top; ++k) a += gt[r * gts + k];
    const A h = u ? u[r * us] : (A)0;
    if (u) a += h * entropy[r * es];
    const int k = threadIdx.x;
    if (k < n_top) {
      const int64_t j = top[r * ps + k];
      id[k] = j >= 0 && j < cols ? (int)j : -1;
      val[k] = gt[r * gts + k] * inv_t;
    }
    if (k == n_top) {
      id[k] = g && t >= 0 && t < cols ? (int)t : -1;
      val[k] = w * inv_t;
    }
    return {st[0], st[1], -a * inv_t, -h * (A)kLn2 * inv_t};
  }
};

template <class A>
struct KdGrad {
  enum { kEntries = THX_MAX_TEACHER };
  Teacher<A> t;
  const A* stats; int64_t ss;
  const A* g; int64_t gs;
  A c, temperature;

  THX_DEV int entries() const { return t.n; }
  THX_DEV Slope<A> open(int64_t r, int64_t cols, int* id, A* val) const {
    const A* st = stats + r * ss;
    const A tm = st[2], tls = st[3], gt = g[r * gs] * temperature;
    const bool tnone = tm == neg_inf<A>() && tls == neg_inf<A>();
    for (int k = threadIdx.x; k < t.n; k += blockDim.x) {
      const int64_t j = load_index(t.ids, t.i64, r * t.is + k);
      id[k] = j >= 0 && j < cols && !tnone ? (int)j : -1;
      val[k] = -gt * acc_exp2((load_real<A>(t.logits, t.dtype, r * t.ls + k) - tm) * c - tls);
    }
    return {st[0], st[1], tls != tls ? tls : tnone ? (A)0 : gt, (A)0};
  }
};

template <class T, bool FUSED>
struct GradCut {
  typedef typename AccOf<T>::type A;
  const T* x;
  int64_t xs, rows, cols;
  int64_t per;  // vectors of a segment
  int segs;     // segments of a row
  Exponents<T, FUSED> ex;
  T* dx;
  bool nt;      // dx is streamed past the caches
};


// The slope of a row's elements.
template <class T, bool FUSED>
struct RowSlope {
  typedef typename AccOf<T>::type A;
  Exponents<T, FUSED> ex;
  A ref, a, b;
  bool none;
  THX_DEV RowSlope(const Slope<A>& s, const Exponents<T, FUSED>& ex_) : ex(ex_) {
    none = s.m == neg_inf<A>() && s.ls == neg_inf<A>();
    ref = ex.reference(s.m);
    const A inv = none ? (A)0 : acc_exp2(-s.ls);
    a = none ? (A)0 : (s.a - s.b * s.ls) * inv;
    b = s.b * inv;
  }
  THX_DEV A operator()(T v) const { return b == (A)0 ? of<false>(v) : of<true>(v); }
  template <bool B>
  THX_DEV A of(T v) const {
    const A d = ex.of((A)v, ref), e = acc_exp2(d);
    return B ? e * (a + b * LaneSums<T, false>::bounded(d)) : e * a;
  }
  // In place, over N vectors; whether there is a b is the same for the whole row.
  template <int V, int N>
  THX_DEV void over(Vec<T, V> (&v)[N]) const {
    if (none) {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) v[u].v[e] = (T)0;
    } else if (b == (A)0) {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) v[u].v[e] = (T)of<false>(v[u].v[e]);
    } else {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) v[u].v[e] = (T)of<true>(v[u].v[e]);
    }
  }
};

// Element j of a row's gradient, which entry k of the list names, written over; behind a barrier.  The first entry of a
// column writes for all that name it.
template <class T, class A, bool FUSED>
THX_DEV void write_entry(const RowSlope<T, FUSED>& slope, T at, T* dx, const int* id, const A* val, int n, int k, int j) {
  A v = 0;
  int before = 0, i = 0;
  for (; i + 4 <= n; i += 4) {  // four at a time: each is a wait for LDS
    const int4 o = *(const int4*)(id + i);
    if (o.x == j || o.y == j || o.z == j || o.w == j) {
      v += (o.x == j ? val[i] : (A)0) + (o.y == j ? val[i + 1] : (A)0) + (o.z == j ? val[i + 2] : (A)0) +
           (o.w == j ? val[i + 3] : (A)0);
      before |= (i < k && o.x == j) | (i + 1 < k && o.y == j) | (i + 2 < k && o.z == j) | (i + 3 < k && o.w == j);
    }
  }
  for (; i < n; ++i)
    if (id[i] == j) {
      v += val[i];
      before |= i < k;
    }
  if (!before) dx[j] = (T)(slope(at) + v);
}

// All elements of columns [first, last) that the list names.
template <class T, class A, bool FUSED>
THX_DEV void write_entries(const RowSlope<T, FUSED>& slope, const T* x, T* dx, const int* id, const A* val, int n, int64_t first,
                           int64_t last, int from = 0) {
  for (int k = from + threadIdx.x; k < n; k += blockDim.x) {
    const int j = id[k];
    if (j >= first && j < last) write_entry(slope, x[j], dx, id, val, n, k, j);
  }
}

template <class T, class Row, bool FUSED>
__global__ void __launch_bounds__(256) vocab_grad(GradCut<T, FUSED> q, Row row) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value;
  __shared__ __align__(16) int id[Row::kEntries];
  __shared__ A val[Row::kEntries];
  const int64_t units = q.rows * q.segs, whole = q.cols / V, vectors = (q.cols + V - 1) / V;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t r = unit / q.segs, seg = unit - r * q.segs;
    const T* x = q.x + r * q.xs;
    T* dx = q.dx + r * q.cols;
    const RowSlope<T, FUSED> slope(row.open(r, q.cols, id, val), q.ex);
    const int64_t lo = seg * q.per, hi = lo + q.per < vectors ? lo + q.per : vectors;
    for (int64_t i0 = lo; i0 < hi; i0 += 256 * kUnroll) {
      Vec<T, V> v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = i0 + u * 256 + threadIdx.x;
        if (i < hi && i < whole) load_vec<T, V, false, true>(v[u], x + i * V);
      }
      slope.over(v);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = i0 + u * 256 + threadIdx.x;
        if (i < hi && i < whole) {
          store_out(dx + i * V, v[u], q.nt);
        } else if (i < hi) {
          for (int64_t j = i * V; j < q.cols; ++j) dx[j] = slope.none ? (T)0 : (T)slope(x[j]);
        }
      }
    }
    __syncthreads();  // the entries are there, and the elements they replace are written
    if (!slope.none) write_entries(slope, x, dx, id, val, row.entries(), lo * V, hi * V);
    __syncthreads();  // before the next row's entries
  }
}

// ---- forward and gradient in one ---------------------------------------------------------------------------------------
//
// Where the gradients of a row's results are known beforehand (the weight of a loss), one block reads the row once, keeps
// it in registers through the sums, and writes the gradient from there: two passes over memory instead of three.

template <class T>
struct LpTrain {
  typedef typename AccOf<T>::type A;
  enum { kEntries = 1, kEntropy = 1 };
  LpRow<T> out;
  const A* g; int64_t gs;
  const A* u; int64_t us;
};

template <class T>
struct KdTrain {
  typedef typename AccOf<T>::type A;
  enum { kEntries = THX_MAX_TEACHER, kEntropy = 0 };
  KdRow<T> out;
  const A* g; int64_t gs;
  A temperature;
};

template <class T, class Row, int THREADS, int VPT, bool FUSED>
__global__ void __launch_bounds__(THREADS, VPT > 8 && sizeof(T) < 8 ? 4 : 1) vocab_train(GradCut<T, FUSED> q, Row row) {
  typedef typename AccOf<T>::type A;
  constexpr int V = Width<T>::value, W = THREADS / 64;
  constexpr bool ENT = Row::kEntropy;
  constexpr int G = VPT % 4 ? (VPT % 2 ? 1 : 2) : 4;  // vectors between two looks at the maximum
  __shared__ __align__(16) int id[Row::kEntries];
  __shared__ A val[Row::kEntries];
  __shared__ A part[W][ENT ? 3 : 4], losses[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  // rounds that every thread takes part in, and the vectors and elements that are left
  const int whole = (int)(q.cols / V), full = whole / THREADS, rest = (int)(q.cols - (int64_t)whole * V);
  for (int64_t r = blockIdx.x; r < q.rows; r += gridDim.x) {
    const T* x = q.x + r * q.xs;
    T* dx = q.dx + r * q.cols;
    const T* xt = x + (int)threadIdx.x * V;
    // a teacher's entry to each thread, on its way before the row: what hangs on it is not waited for behind the row
    [[maybe_unused]] int mine_id = -1;  // the row's length where it names a column that is not there
    [[maybe_unused]] A mine_logit = neg_inf<A>();
    [[maybe_unused]] T mine_at = (T)0;
    if constexpr (!ENT) {
      if ((int)threadIdx.x < row.out.t.n) {
        const Entry<A> e = load_entry(row.out.t, r, threadIdx.x);
        mine_id = (int)(e.id < 0 ? -1 : e.id < q.cols ? e.id : q.cols), mine_logit = e.logit;
      }
    }
    Vec<T, V> v[VPT];
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      if (u < full) {
        load_vec<T, V, false, true>(v[u], xt + u * (THREADS * V));
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u].v[e] = (T)neg_inf<A>();
        if (u == full && u * THREADS + (int)threadIdx.x < whole) load_vec<T, V, false, true>(v[u], xt + u * (THREADS * V));
      }
    }
    // the elements behind the last whole vector, one to a thread
    const bool extra = (int)threadIdx.x < rest;
    const T tail = extra ? x[(int64_t)whole * V + threadIdx.x] : (T)neg_inf<A>();
    if constexpr (!ENT) mine_at = entry_at<T, A>({mine_id, mine_logit}, x, q.cols);
    LaneSums<T, ENT, FUSED> sum;
    sum.init();
    if ((A)tail > sum.m) sum.raise((A)tail, q.ex);
    sum.add((A)tail, q.ex);
#pragma unroll
    for (int u = 0; u < VPT; u += G) {
      if (u > full) continue;
      A m = vector_max(v[u]);
#pragma unroll
      for (int k = 1; k < G; ++k) {
        const A o = vector_max(v[u + k]);
        m = m > o ? m : o;
      }
      if (m > sum.m) sum.raise(m, q.ex);
#pragma unroll
      for (int k = 0; k < G; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum.add((A)v[u + k].v[e], q.ex);
    }
#pragma unroll
    for (int u = 0; u < VPT; ++u) forget(v[u]);
    sum.join_lanes(q.ex);
    if (lane == 0) {
      part[wave][0] = sum.m, part[wave][1] = sum.s;
      if constexpr (ENT) part[wave][2] = sum.w;
    }
    [[maybe_unused]] LaneSums<A, false> ts;
    [[maybe_unused]] const Exponents<A> tex = {q.ex.c};
    if constexpr (!ENT) {
      ts.init();
      take_entry({mine_id, mine_logit}, q.cols, tex, ts);
      for (int k = threadIdx.x + THREADS; k < row.out.t.n; k += THREADS)
        take_entry(load_entry(row.out.t, r, k), q.cols, tex, ts);
      ts.join_lanes(tex);
      if (lane == 0) part[wave][2] = ts.m, part[wave][3] = ts.s;
    }
    __syncthreads();
    sum.init();
    if constexpr (!ENT) ts.init();
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum.join(part[w][0], part[w][1], ENT ? part[w][2] : (A)0, q.ex);
      if constexpr (!ENT) ts.join(part[w][2], part[w][3], (A)0, tex);
    }
    const A ls = sum.log2_sum();
    Slope<A> s = {sum.m, ls, (A)0, (A)0};
    int n;
    [[maybe_unused]] A tls, gt;
    if constexpr (ENT) {
      const LpRow<T>& o = row.out;
      n = 1;
      const int64_t t = load_index(o.tokens, o.t64, r * o.ts);
      const A w = row.g && t >= 0 ? row.g[r * row.gs] : (A)0, h = row.u ? row.u[r * row.us] : (A)0;
      const A entropy = sum.nothing_left() ? (A)0 : (ls - sum.w / sum.s) * (A)kLn2;
      s.a = -((t >= q.cols && row.g ? (A)NAN : w) + (row.u ? h * entropy : (A)0)) * o.inv_t;
      s.b = -h * (A)kLn2 * o.inv_t;
      if (threadIdx.x == 0) {
        id[0] = row.g && t >= 0 && t < q.cols ? (int)t : -1;
        val[0] = w * o.inv_t;
        A lp = 0;
        if (t >= q.cols) lp = (A)NAN;
        else if (t >= 0) lp = sum.nothing_left() ? neg_inf<A>() : q.ex.log_prob((A)x[t], sum.m, o.inv_t, ls);
        o.o.log_prob[r] = lp;
        o.o.entropy[r] = entropy;
        o.o.stats[2 * r] = sum.m;
        o.o.stats[2 * r + 1] = ls;
      }
    } else {
      const KdRow<T>& o = row.out;
      n = o.t.n;
      tls = ts.log2_sum(), gt = row.g[r * row.gs] * row.temperature;
      s.a = tls != tls ? tls : ts.nothing_left() ? (A)0 : gt;
      if (threadIdx.x == 0) {
        o.stats[4 * r] = sum.m;
        o.stats[4 * r + 1] = ls;
        o.stats[4 * r + 2] = ts.m;
        o.stats[4 * r + 3] = tls;
      }
    }
    const RowSlope<T, FUSED> slope(s, q.ex);
    T* dt = dx + (int)threadIdx.x * V;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      if (u > full) continue;
      Vec<T, V> o[1] = {v[u]};
      slope.over(o);
      if (u < full || u * THREADS + (int)threadIdx.x < whole) store_out(dt + u * (THREADS * V), o[0], q.nt);
    }
    if (extra) dx[(int64_t)whole * V + threadIdx.x] = slope.none ? (T)0 : (T)slope(tail);
    if constexpr (!ENT) {  // behind the stores: the registers that held the row are free
      const KdRow<T>& o = row.out;
      A loss = 0;
      auto put = [&](int k, const Entry<A>& e, T at) {
        id[k] = e.id >= 0 && e.id < q.cols && !ts.nothing_left() ? (int)e.id : -1;
        val[k] = -gt * acc_exp2(tex.of(e.logit, ts.m) - tls);
        loss += entry_loss(o, e, at, q.cols, q.ex, sum, ls, ts.m, tls);
      };
      if ((int)threadIdx.x < n) put(threadIdx.x, {mine_id, mine_logit}, mine_at);
      for (int k = threadIdx.x + THREADS; k < n; k += THREADS) {
        const Entry<A> e = load_entry(o.t, r, k);
        put(k, e, entry_at(e, x, q.cols));
      }
      loss = lanes_sum<64>(loss);
      if (lane == 0) losses[wave] = loss;
    }
    __syncthreads();  // the entries and the losses are there, and the elements that the entries replace are written
    if constexpr (ENT) {
      if (!slope.none) write_entries(slope, x, dx, id, val, n, 0, q.cols);
    } else {
      if (!slope.none) {
        const int j = (int)threadIdx.x < n ? id[threadIdx.x] : -1;
        if (j >= 0) write_entry(slope, mine_at, dx, id, val, n, threadIdx.x, j);
        write_entries(slope, x, dx, id, val, n, 0, q.cols, THREADS);
      }
      if (threadIdx.x == 0) {
        A loss = losses[0];
        for (int w = 1; w < W; ++w) loss += losses[w];
        row.out.loss[r] = (sum.s != sum.s ? sum.s : loss) * row.out.t2;
      }
    }
    __syncthreads();  // before the next row's
  }
}

int acc_code(int dtype) { return dtype == THX_F64 ? THX_F64 : THX_F32; }
bool is_float(int dtype) { return dtype == THX_F16 || dtype == THX_F32 || dtype == THX_F64; }
unsigned grid_of(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(n, 1 << 20)); }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a call's rows are cut for the forward pass: enough waves to fill the device, one per row where there are rows enough
// (nothing to join then), and no more than 64 parts, each of at least one step of a wave.
int parts_of(int64_t rows, int64_t vectors) {
  const int64_t want = ceil_div((int64_t)compute_units() * 16, std::max<int64_t>(rows, 1));
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, 64, ceil_div(vectors, 64)}));
}

// Sums, then lists, of all parts.
size_t partial_bytes(const Rows& x, int n_top) {
  const int isz = dtype_size(x.dtype);
  const int64_t parts = parts_of(x.rows, ceil_div(x.cols * isz, 16));
  if (parts == 1 || !x.rows) return 0;
  const int acc = dtype_size(acc_code(x.dtype));
  const size_t sums = ((size_t)x.rows * parts * 3 * acc + 15) / 16 * 16;
  return sums + (size_t)x.rows * parts * n_top * (acc == 8 ? 16 : 8);
}

std::string plan_of(const char* name, const Rows& x) {
  return std::string(name) + "|t" + std::to_string(x.dtype) + "|p" +
         std::to_string(parts_of(x.rows, ceil_div(x.cols * dtype_size(x.dtype), 16)));
}

// f(T(), whether the exponents are the fused ones) for the type of the logits.
template <class F>
int by_type(int x, double temperature, F&& f) {
  if (x == THX_F16) {
    // the largest finite half times c below 2^24
    if (65504.0 * (kLog2E / temperature) < 16777216.0) return f(thx_f16(), std::true_type());
    return f(thx_f16(), std::false_type());
  }
  if (x == THX_F32) return f(thx_f32(), std::false_type());
  return f(thx_f64(), std::false_type());
}

template <class T, bool FUSED>
Cut<T, FUSED> cut_of(const Rows& x, double temperature, void* ws) {
  typedef typename AccOf<T>::type A;
  Cut<T, FUSED> q;
  const int64_t vectors = ceil_div(x.cols, Width<T>::value);
  q.x = (const T*)x.ptr;
  q.xs = x.stride, q.rows = x.rows, q.cols = x.cols;
  q.parts = parts_of(x.rows, vectors);
  q.per = ceil_div(vectors, q.parts);
  q.ex = {(A)(kLog2E / temperature)};
  q.partial = (A*)ws;
  q.lists = (typename Order<T>::Key*)((char*)ws + ((size_t)x.rows * q.parts * 3 * sizeof(A) + 15) / 16 * 16);
  return q;
}

template <class T, bool TOP, bool ENT, bool FUSED, class Row>
int launch_forward(Cut<T, FUSED> q, Row row, const std::string& plan) {
  void* args[] = {&q, &row};
  const int64_t units = q.rows * q.parts;
  int rc = launch_builtin((const void*)&vocab_read<T, TOP, Row, ENT, FUSED>, plan, dim3(grid_of(ceil_div(units, kWaves))),
                          dim3(64 * kWaves), args);
  if (rc || q.parts == 1) return rc;
  return launch_builtin((const void*)&vocab_join<T, TOP, Row, ENT, FUSED>, plan + "|join", dim3(grid_of(q.rows)), dim3(64), args);
}

// The gradient's segments: 16 blocks to a compute unit where there are too few rows for that, one vector to a thread at
// least; whole rows else, since every segment reads the row's list again (2048 rows of 32000 floats, 64 entries: 153 us
// in segments of 4 vectors to a thread, 116 us in two segments a row).
template <class T, bool FUSED, class Row>
int launch_grad(const Rows& x, double temperature, const Rows& dx, Row row, const std::string& plan) {
  typedef typename AccOf<T>::type A;
  GradCut<T, FUSED> q;
  const int64_t vectors = ceil_div(x.cols, Width<T>::value);
  q.x = (const T*)x.ptr;
  q.xs = x.stride, q.rows = x.rows, q.cols = x.cols;
  q.segs = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(vectors, 256), ceil_div(16 * compute_units(), x.rows)));
  q.per = ceil_div(vectors, q.segs);
  q.ex = {(A)(kLog2E / temperature)};
  q.dx = (T*)dx.ptr;
  q.nt = stream_out(x, dx);
  void* args[] = {&q, &row};
  return launch_builtin((const void*)&vocab_grad<T, Row, FUSED>, plan, dim3(grid_of(x.rows * q.segs)), dim3(256), args);
}

// The block that holds a row of the one-pass kernel: threads, and vectors to a thread; 0 where none does.  Two blocks of a
// compute unit hide each other's waits, so 512 threads with up to 20 vectors (no more than 128 registers) come before 1024:
// 4877 rows of 50257 halves in 512x16 211 us, in 1024x8 215 (228 and 254 with 64 teacher's entries, where 64 registers do
// not do); 3000 rows of 80000 in 512x20 200 us, in 1024x16 240.  Up to 4096 vectors 8 to a thread leave room for four
// blocks: 8192 rows of 32000 halves in 512x8 192 us, in 256x16 210.  Doubles take a third more registers, and no more than
// 8192 vectors.
struct Hold {
  int threads = 0, vpt = 0;
};
Hold hold_of(const Rows& x) {
  static const Hold all[] = {{256, 1}, {256, 2}, {256, 4}, {256, 8}, {512, 8}, {512, 16}, {512, 20}, {1024, 16}, {1024, 20}};
  const int isz = dtype_size(x.dtype);
  const int64_t whole = x.cols / (16 / isz);  // the elements behind the last whole vector go to one thread each
  for (const Hold& h : all)
    if (whole <= (int64_t)h.threads * h.vpt && !(isz == 8 && h.vpt * h.threads > 8192)) return h;
  return Hold();
}

std::string held_plan(const char* name, const Rows& x, const Hold& h) {
  return std::string(name) + "|t" + std::to_string(x.dtype) + "|r" + std::to_string(h.threads) + "x" + std::to_string(h.vpt);
}

template <class T, bool FUSED, class Row>
int launch_train(const Rows& x, double temperature, const Rows& dx, const Hold& h, Row row, const std::string& plan) {
  typedef typename AccOf<T>::type A;
  GradCut<T, FUSED> q = {};
  q.x = (const T*)x.ptr;
  q.xs = x.stride, q.rows = x.rows, q.cols = x.cols;
  q.ex = {(A)(kLog2E / temperature)};
  q.dx = (T*)dx.ptr;
  q.nt = stream_out(x, dx);
  void* args[] = {&q, &row};
  const void* kernel = nullptr;
  switch (h.threads * 32 + h.vpt) {
    case 256 * 32 + 1: kernel = (const void*)&vocab_train<T, Row, 256, 1, FUSED>; break;
    case 256 * 32 + 2: kernel = (const void*)&vocab_train<T, Row, 256, 2, FUSED>; break;
    case 256 * 32 + 4: kernel = (const void*)&vocab_train<T, Row, 256, 4, FUSED>; break;
    case 256 * 32 + 8: kernel = (const void*)&vocab_train<T, Row, 256, 8, FUSED>; break;
    case 512 * 32 + 8: kernel = (const void*)&vocab_train<T, Row, 512, 8, FUSED>; break;
    case 512 * 32 + 16: kernel = (const void*)&vocab_train<T, Row, 512, 16, FUSED>; break;
    default:
      if constexpr (sizeof(T) < 8)
        kernel = h.threads == 512  ? (const void*)&vocab_train<T, Row, 512, 20, FUSED>
                 : h.vpt == 16 ? (const void*)&vocab_train<T, Row, 1024, 16, FUSED>
                               : (const void*)&vocab_train<T, Row, 1024, 20, FUSED>;
  }
  return launch_builtin(kernel, plan, dim3(grid_of(x.rows)), dim3(h.threads), args);
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

// The gradient of a result with one value per row: such values, or one value (every extent 1) for all rows.
int row_gradient(const char* what, const char* name, const thx_array* a, const thx_array* x, int acc, int flags, Rows* r) {
  bool one = a->nd == x->nd - 1;
  for (int d = 0; one && d < a->nd; ++d) one = a->shape[d] == 1;
  if (!one) return like_rows(what, name, a, x, acc, -1, flags, r);
  int rc = rows_of(what, name, a, acc, 0, flags, r);
  r->stride = 0;
  return rc;
}

int token_logprob(const thx_array* logits, const thx_array* tokens, double temperature, int n_top, const thx_array* log_prob,
                  const thx_array* entropy, const thx_array* top, const thx_array* top_at, const thx_array* stats, void* ws,
                  size_t ws_bytes, int flags) {
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
  if ((rc = check_workspace(what, ws, ws_bytes, partial_bytes(in[0], n_top), flags))) return rc;
  const std::string plan = plan_of("lp", in[0]) + (n_top ? "|top" : "");
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, temperature, [&](auto t, auto fused) {
    typedef decltype(t) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const LpRow<T> row = {in[1].ptr, in[1].stride, in[1].dtype == THX_I64, n_top, (A)(1.0 / temperature),
                          {(A*)out[0].ptr, (A*)out[1].ptr, (A*)out[3].ptr, (int64_t*)out[4].ptr, (A*)out[2].ptr}};
    const Cut<T, FUSED> q = cut_of<T, FUSED>(in[0], temperature, ws);
    return n_top ? launch_forward<T, true, true>(q, row, plan) : launch_forward<T, false, true>(q, row, plan);
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
  if (g && (rc = row_gradient(what, "g_log_prob", g, logits, acc, flags, &in[5]))) return rc;
  if (u && (rc = row_gradient(what, "g_entropy", u, logits, acc, flags, &in[6]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, in[0].dtype, in[0].cols, flags, &out))) return rc;
  if ((rc = contiguous_rows(what, "dlogits", out))) return rc;
  if ((rc = no_overlap(what, &out, 1, in, 8)) && !dry) return rc;
  const std::string plan = "lpg|t" + std::to_string(in[0].dtype);
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, temperature, [&](auto t, auto fused) {
    typedef decltype(t) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const LpGrad<A> q = {in[1].ptr, in[1].stride, in[1].dtype == THX_I64, (const A*)in[2].ptr, in[2].stride, (const A*)in[3].ptr,
                   in[3].stride, (const int64_t*)in[4].ptr, in[4].stride, (int)n_top, (const A*)in[5].ptr, in[5].stride,
                   (const A*)in[6].ptr, in[6].stride, (const A*)in[7].ptr, in[7].stride, (A)(1.0 / temperature)};
    return launch_grad<T, FUSED>(in[0], temperature, out, q, plan);
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
                 const thx_array* loss, const thx_array* stats, void* ws, size_t ws_bytes, int flags) {
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
  if ((rc = check_workspace(what, ws, ws_bytes, partial_bytes(in[0], 0), flags))) return rc;
  const std::string plan = plan_of("kd", in[0]);
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, temperature, [&](auto t, auto fused) {
    typedef decltype(t) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const KdRow<T> row = {teacher_args<A>(in[1], in[2]), (A)(1.0 / temperature), (A)(temperature * temperature),
                          (A*)out[0].ptr, (A*)out[1].ptr};
    return launch_forward<T, false, false>(cut_of<T, FUSED>(in[0], temperature, ws), row, plan);
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
  if ((rc = !g ? fail(THX_ERR_ARG, "%s: g_loss is missing", what) : row_gradient(what, "g_loss", g, logits, acc, flags, &in[4]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, in[0].dtype, in[0].cols, flags, &out))) return rc;
  if ((rc = contiguous_rows(what, "dlogits", out))) return rc;
  if ((rc = no_overlap(what, &out, 1, in, 5)) && !dry) return rc;
  const std::string plan = "kdg|t" + std::to_string(in[0].dtype);
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(in[0].dtype, temperature, [&](auto t, auto fused) {
    typedef decltype(t) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const KdGrad<A> row = {teacher_args<A>(in[1], in[2]), (const A*)in[3].ptr, in[3].stride, (const A*)in[4].ptr,
                           in[4].stride, (A)(kLog2E / temperature), (A)temperature};
    return launch_grad<T, FUSED>(in[0], temperature, out, row, plan);
  });
}

int token_logprob_train(const thx_array* logits, const thx_array* tokens, const thx_array* g, const thx_array* u,
                        double temperature, const thx_array* log_prob, const thx_array* entropy, const thx_array* stats,
                        const thx_array* dx, void* ws, size_t ws_bytes, int flags) {
  const char* what = "token log probabilities with their gradient";
  // the checks, and the two calls where no block holds a row
  int rc = token_logprob(logits, tokens, temperature, 0, log_prob, entropy, nullptr, nullptr, stats, ws, ws_bytes,
                         flags | THX_DRY_RUN);
  if (!rc) rc = token_logprob_grad(logits, tokens, stats, entropy, nullptr, g, u, nullptr, temperature, dx, flags | THX_DRY_RUN);
  if (rc) return rc;
  Rows x, t, gr, ur, out[4];
  if ((rc = logits_of(what, logits, temperature, flags, &x))) return rc;
  const Hold h = hold_of(x);
  if (!h.threads) {
    rc = token_logprob(logits, tokens, temperature, 0, log_prob, entropy, nullptr, nullptr, stats, ws, ws_bytes, flags);
    return rc ? rc : token_logprob_grad(logits, tokens, stats, entropy, nullptr, g, u, nullptr, temperature, dx, flags);
  }
  const int acc = acc_code(x.dtype);
  if ((rc = indices_of(what, "tokens", tokens, logits, -1, flags, &t))) return rc;
  if (g && (rc = row_gradient(what, "g_log_prob", g, logits, acc, flags, &gr))) return rc;
  if (u && (rc = row_gradient(what, "g_entropy", u, logits, acc, flags, &ur))) return rc;
  if ((rc = like_rows(what, "log_prob", log_prob, logits, acc, -1, flags, &out[0]))) return rc;
  if ((rc = like_rows(what, "entropy", entropy, logits, acc, -1, flags, &out[1]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 2, flags, &out[2]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, x.dtype, x.cols, flags, &out[3]))) return rc;
  const Rows ins[] = {x, t, gr, ur};
  if ((rc = no_overlap(what, out, 4, ins, 4)) && !(flags & THX_DRY_RUN)) return rc;
  const std::string plan = held_plan("lpt", x, h);
  set_last_plan(plan);
  if ((flags & THX_DRY_RUN) || !x.rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(x.dtype, temperature, [&](auto tag, auto fused) {
    typedef decltype(tag) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const LpTrain<T> row = {{t.ptr, t.stride, t.dtype == THX_I64, 0, (A)(1.0 / temperature),
                             {(A*)out[0].ptr, (A*)out[1].ptr, nullptr, nullptr, (A*)out[2].ptr}},
                            (const A*)gr.ptr, gr.stride, (const A*)ur.ptr, ur.stride};
    return launch_train<T, FUSED>(x, temperature, out[3], h, row, plan);
  });
}

int topk_distill_train(const thx_array* logits, const thx_array* teacher, const thx_array* tokens, const thx_array* g,
                       double temperature, const thx_array* loss, const thx_array* stats, const thx_array* dx, void* ws,
                       size_t ws_bytes, int flags) {
  const char* what = "distillation loss with its gradient";
  int rc = topk_distill(logits, teacher, tokens, temperature, loss, stats, ws, ws_bytes, flags | THX_DRY_RUN);
  if (!rc) rc = topk_distill_grad(logits, teacher, tokens, stats, g, temperature, dx, flags | THX_DRY_RUN);
  if (rc) return rc;
  Rows x, t, ids, gr, out[3];
  if ((rc = logits_of(what, logits, temperature, flags, &x))) return rc;
  const Hold h = hold_of(x);
  if (!h.threads) {
    rc = topk_distill(logits, teacher, tokens, temperature, loss, stats, ws, ws_bytes, flags);
    return rc ? rc : topk_distill_grad(logits, teacher, tokens, stats, g, temperature, dx, flags);
  }
  const int acc = acc_code(x.dtype);
  if ((rc = teacher_of(what, teacher, tokens, logits, flags, &t, &ids))) return rc;
  if ((rc = row_gradient(what, "g_loss", g, logits, acc, flags, &gr))) return rc;
  if ((rc = like_rows(what, "loss", loss, logits, acc, -1, flags, &out[0]))) return rc;
  if ((rc = like_rows(what, "stats", stats, logits, acc, 4, flags, &out[1]))) return rc;
  if ((rc = like_rows(what, "dlogits", dx, logits, x.dtype, x.cols, flags, &out[2]))) return rc;
  const Rows ins[] = {x, t, ids, gr};
  if ((rc = no_overlap(what, out, 3, ins, 4)) && !(flags & THX_DRY_RUN)) return rc;
  const std::string plan = held_plan("kdt", x, h);
  set_last_plan(plan);
  if ((flags & THX_DRY_RUN) || !x.rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_type(x.dtype, temperature, [&](auto tag, auto fused) {
    typedef decltype(tag) T;
    constexpr bool FUSED = decltype(fused)::value;
    typedef typename AccOf<T>::type A;
    const KdTrain<T> row = {{teacher_args<A>(t, ids), (A)(1.0 / temperature), (A)(temperature * temperature),
                             (A*)out[0].ptr, (A*)out[1].ptr},
                            (const A*)gr.ptr, gr.stride, (A)temperature};
    return launch_train<T, FUSED>(x, temperature, out[2], h, row, plan);
  });
}

int workspace_of(const char* what, const thx_array* logits, int n_top, size_t* nbytes) {
  if (!logits || !nbytes) return fail(THX_ERR_ARG, "%s: null argument", what);
  if (n_top < 0 || n_top > THX_MAX_TOP) return fail(THX_ERR_ARG, "%s: %d alternatives (at most %d)", what, n_top, THX_MAX_TOP);
  Rows r;
  int rc = logits_of(what, logits, 1.0, THX_DRY_RUN, &r);
  if (!rc) *nbytes = partial_bytes(r, n_top);
  return rc;
}

}  // namespace
}  // namespace thx

using namespace thx;

extern "C" {

int thx_token_logprob_workspace(const thx_array* logits, int n_top, size_t* nbytes) {
  return guarded("thx_token_logprob_workspace", [&] {
    return workspace_of("thx_token_logprob_workspace", logits, n_top, nbytes);
  });
}

int thx_token_logprob_call(const thx_array* logits, const thx_array* tokens, double temperature, int n_top,
                           const thx_array* log_prob, const thx_array* entropy, const thx_array* top_log_probs,
                           const thx_array* top_tokens, const thx_array* stats, void* workspace,
                           size_t workspace_bytes, int flags) {
  return guarded("thx_token_logprob_call", [&] {
    return token_logprob(logits, tokens, temperature, n_top, log_prob, entropy, top_log_probs, top_tokens, stats, workspace,
                         workspace_bytes, flags);
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
    return workspace_of("thx_topk_distill_workspace", logits, 0, nbytes);
  });
}

int thx_topk_distill_call(const thx_array* logits, const thx_array* teacher, const thx_array* tokens, double temperature,
                          const thx_array* loss, const thx_array* stats, void* workspace, size_t workspace_bytes,
                          int flags) {
  return guarded("thx_topk_distill_call",
                 [&] { return topk_distill(logits, teacher, tokens, temperature, loss, stats, workspace, workspace_bytes, flags); });
}

int thx_topk_distill_grad_call(const thx_array* logits, const thx_array* teacher, const thx_array* tokens,
                               const thx_array* stats, const thx_array* g_loss, double temperature,
                               const thx_array* dlogits, int flags) {
  return guarded("thx_topk_distill_grad_call",
                 [&] { return topk_distill_grad(logits, teacher, tokens, stats, g_loss, temperature, dlogits, flags); });
}

int thx_token_logprob_train_call(const thx_array* logits, const thx_array* tokens, const thx_array* g_log_prob,
                                 const thx_array* g_entropy, double temperature, const thx_array* log_prob,
                                 const thx_array* entropy, const thx_array* stats, const thx_array* dlogits,
                                 void* workspace, size_t workspace_bytes, int flags) {
  return guarded("thx_token_logprob_train_call", [&] {
    return token_logprob_train(logits, tokens, g_log_prob, g_entropy, temperature, log_prob, entropy, stats, dlogits,
                               workspace, workspace_bytes, flags);
  });
}

int thx_topk_distill_train_call(const thx_array* logits, const thx_array* teacher, const thx_array* tokens,
                                const thx_array* g_loss, double temperature, const thx_array* loss,
                                const thx_array* stats, const thx_array* dlogits, void* workspace,
                                size_t workspace_bytes, int flags) {
  return guarded("thx_topk_distill_train_call", [&] {
    return topk_distill_train(logits, teacher, tokens, g_loss, temperature, loss, stats, dlogits, workspace,
                              workspace_bytes, flags);
  });
}

}  // extern "C"
