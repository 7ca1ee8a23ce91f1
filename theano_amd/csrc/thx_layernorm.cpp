// Layer normalisation over rows and its gradients: planner and kernels.
#include "thx_rows.h"

#include "kernels/thx_common.h"

namespace thx {
namespace {

template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

template <class A>
THX_DEV A block_sum(A v, A* lds) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  A r = lds[0];
  for (unsigned w = 1; w < blockDim.x / 64; ++w) r += lds[w];
  return r;
}

template <class T, class P>
__global__ void __launch_bounds__(256) ln_forward(const T* x, int64_t xs, int64_t rows, int64_t cols, const P* gamma, int64_t gs,
                                                  const P* beta, int64_t bs, double eps, T* y,
                                                  typename AccOf<T>::type* mean, typename AccOf<T>::type* invstd) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[4];
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
__global__ void __launch_bounds__(256) ln_grad_rows(const T* x, int64_t xs, const T* dy, int64_t ds, int64_t rows, int64_t cols,
                                                    const P* gamma, int64_t gs, const typename AccOf<T>::type* mean,
                                                    int64_t ms, const typename AccOf<T>::type* invstd, int64_t is, T* dx) {
  typedef typename AccOf<T>::type A;
  __shared__ A lds[4];
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
__global__ void __launch_bounds__(256) ln_grad_params(const T* x, int64_t xs, const T* dy, int64_t ds, int64_t rows,
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

template <class A, class P>
__global__ void __launch_bounds__(256) ln_grad_join(const A* partial, int slices, int64_t cols, P* dgamma, P* dbeta) {
  for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < cols; c += (int64_t)gridDim.x * blockDim.x) {
    A g = 0, b = 0;
    for (int s = 0; s < slices; ++s) {
      g += partial[(int64_t)s * 2 * cols + c];
      b += partial[((int64_t)s * 2 + 1) * cols + c];
    }
    if (dgamma) dgamma[c] = (P)g;
    if (dbeta) dbeta[c] = (P)b;
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

int slices_of(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(64, rows / 64)); }

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
  const std::string plan = "ln|rows";
  set_last_plan(plan);
  if (dry || !in[0].rows) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_types(in[0].dtype, pt, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    void* args[] = {&in[0].ptr, &in[0].stride, &in[0].rows, &in[0].cols, &in[1].ptr, &in[1].stride, &in[2].ptr,
                    &in[2].stride, &epsilon, &out[0].ptr, &out[1].ptr, &out[2].ptr};
    return launch_builtin((const void*)&ln_forward<T, P>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
  });
}

int layernorm_grad_bytes(const thx_array* x, const thx_array* dgamma, size_t* nbytes) {
  if (!x || !nbytes) return fail(THX_ERR_ARG, "layer normalization gradient: null argument");
  Rows r;
  int rc = rows_of("layer normalization gradient", "x", x, -1, 1, THX_DRY_RUN, &r);
  if (rc) return rc;
  *nbytes = dgamma ? (size_t)slices_of(r.rows) * 2 * r.cols * dtype_size(acc_code(r.dtype)) : 0;
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
  const std::string plan = "lng|rows";
  set_last_plan(plan);
  if (dry) return THX_OK;
  if ((rc = ensure_init())) return rc;
  return by_types(in[0].dtype, pt, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    typedef typename AccOf<T>::type A;
    int rc = THX_OK;
    if (in[0].rows && in[0].cols) {
      void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[4].ptr,
                      &in[4].stride, &in[2].ptr, &in[2].stride, &in[3].ptr, &in[3].stride, &out[0].ptr};
      rc = launch_builtin((const void*)&ln_grad_rows<T, P>, plan, dim3(grid_of(in[0].rows)), dim3(256), args);
    }
    if (rc || !dgamma || !in[0].cols) return rc;
    int slices = slices_of(in[0].rows);
    const unsigned blocks = grid_of((in[0].cols + 255) / 256);
    void* args[] = {&in[0].ptr, &in[0].stride, &in[1].ptr, &in[1].stride, &in[0].rows, &in[0].cols, &in[2].ptr,
                    &in[2].stride, &in[3].ptr, &in[3].stride, &ws};
    rc = launch_builtin((const void*)&ln_grad_params<T>, plan, dim3(blocks, slices), dim3(256), args);
    if (rc) return rc;
    void* join[] = {&ws, &slices, &in[0].cols, &out[1].ptr, &out[2].ptr};
    return launch_builtin((const void*)&ln_grad_join<A, P>, plan, dim3(blocks), dim3(256), join);
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

}  // extern "C"
