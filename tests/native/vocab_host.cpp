// The kernels over a vocabulary (theano_amd/csrc/thx_vocab.cpp) on the host: the best columns of rows of many kinds, for
// every type, exponent form and number of parts, against a sort.  VOCAB_KERNELS is the file with the device code.
#include "wave_host.h"

enum { THX_F16 = 9, THX_F32 = 10, THX_F64 = 11, THX_MAX_TOP = 64, THX_MAX_TEACHER = 1024 };
#include VOCAB_KERNELS

#include <numeric>
#include <random>

using namespace thx;

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Arrays of exactly the size that the kernels are promised, ending where the allocation ends.
template <class T>
T* array(size_t n) { return (T*)malloc(std::max<size_t>(1, n * sizeof(T))); }

static int cases = 0, wrong = 0;

template <class T, bool FUSED>
void check(int64_t rows, int64_t cols, int k, int parts, int kind, unsigned seed) {
  typedef typename AccOf<T>::type A;
  typedef typename Order<T>::Key Key;
  std::mt19937 g(seed);
  std::normal_distribution<double> normal;
  T* x = array<T>(rows * cols);
  for (int64_t i = 0; i < rows * cols; ++i) {
    const double v = 3 * normal(g), j = (double)(i % cols);
    const double values[] = {v, (double)(g() % 3), 0, g() % 10 < 6 ? -INFINITY : v, g() % 7 == 0 ? NAN : g() % 11 ? v : INFINITY,
                             -INFINITY, NAN, j / 16, -j / 16, g() % 2 ? 0.0 : -0.0};
    x[i] = (T)values[kind];
  }
  int64_t* tokens = array<int64_t>(rows);
  for (int64_t r = 0; r < rows; ++r) tokens[r] = (int64_t)(g() % (cols + 2)) - 1;
  const int64_t vectors = ceil_div(cols, Width<T>::value);
  const LpRow<T> row = {tokens, 1, 1, k, 1,
                        {array<A>(rows), array<A>(rows), array<A>(rows * k), array<int64_t>(rows * k), array<A>(rows * 2)}};
  Cut<T, FUSED> q;
  q.x = x, q.xs = cols, q.rows = rows, q.cols = cols;
  q.parts = parts, q.per = ceil_div(vectors, parts);
  q.ex = {(A)kLog2E};
  q.partial = parts > 1 ? array<A>(rows * parts * 3) : nullptr;
  q.lists = parts > 1 ? array<Key>(rows * parts * k) : nullptr;
  auto run = [&](auto top) {
    constexpr bool TOP = decltype(top)::value;
    host::launch((unsigned)ceil_div(rows * parts, kWaves), 64 * kWaves, [&] { vocab_read<T, TOP, LpRow<T>, true, FUSED>(q, row); });
    if (parts > 1) host::launch((unsigned)rows, 64, [&] { vocab_join<T, TOP, LpRow<T>, true, FUSED>(q, row); });
  };
  if (k) run(std::true_type());
  else run(std::false_type());
  ++cases;
  for (int64_t r = 0; r < rows; ++r) {
    const T* xr = x + r * cols;
    std::vector<int64_t> at(cols);
    std::iota(at.begin(), at.end(), 0);
    std::stable_sort(at.begin(), at.end(), [&](int64_t a, int64_t b) {
      const double u = (double)xr[a], v = (double)xr[b];
      return u != u || v != v ? u != u && v == v : u > v;
    });
    if (std::equal(at.begin(), at.begin() + k, row.o.top_at + r * k)) continue;
    printf("%d bytes, fused %d, %ld x %ld, %d best, %d parts, kind %d: row %ld\n", (int)sizeof(T), FUSED, (long)rows, (long)cols, k,
           parts, kind, (long)r);
    ++wrong;
  }
  for (void* p : {(void*)x, (void*)tokens, (void*)row.o.log_prob, (void*)row.o.entropy, (void*)row.o.top, (void*)row.o.top_at,
                  (void*)row.o.stats, (void*)q.partial, (void*)q.lists})
    free(p);
}

int main() {
  unsigned seed = 0;
  for (int kind = 0; kind < 10; ++kind)
    for (int64_t cols : {1, 2, 7, 8, 17, 64, 130, 513, 1100, 4097})
      for (int k : {0, 1, 7, 20, 64}) {
        if (cols > 600 && k && k < 20) continue;
        const int best = (int)std::min<int64_t>(k, cols);
        auto each = [&](auto t, auto fused) {
          typedef decltype(t) T;
          const int64_t most = ceil_div(ceil_div(cols, Width<T>::value), 64);   // each part at least one step of a wave
          const int64_t rows = cols == 1100 ? 5 : cols < 100 ? 2 : 1;             // 5: more than the waves of a block
          for (int64_t parts : {(int64_t)1, (int64_t)3, most})
            if (parts <= most) check<T, decltype(fused)::value>(rows, cols, best, (int)parts, kind, ++seed);
        };
        each(thx_f64(), std::false_type());
        each(thx_f32(), std::false_type());
        each(thx_f16(), std::true_type());
        if (kind < 5) each(thx_f16(), std::false_type());
        if (best < k) break;
      }
  printf("%d cases, %d wrong\n", cases, wrong);
  return wrong != 0;
}
