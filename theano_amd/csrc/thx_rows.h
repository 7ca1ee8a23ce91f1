// Host-side helpers of the row operators (thx_layernorm.cpp, thx_vocab.cpp): operands as rows of columns, their
// checks, and the launch of kernels that are compiled into the library.
#pragma once

#include <algorithm>
#include <exception>
#include <new>
#include <string>

#include "thx_internal.h"

namespace thx {

// Nothing thrown may leave through a C entry point.
template <class F>
int guarded(const char* what, F&& body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return fail(THX_ERR_MEMORY, "%s: out of host memory", what);
  } catch (const std::exception& e) {
    return fail(THX_ERR_HIP, "%s: %s", what, e.what());
  } catch (...) {
    return fail(THX_ERR_HIP, "%s: unknown failure", what);
  }
}

// An operand [rows..., cols] (or [rows...], cols = 1): element strides of a row and the address of its first element.
struct Rows {
  char* ptr = nullptr;
  int dtype = 0, nd = 0;
  int64_t rows = 1, cols = 1;
  int64_t stride = 0;              // elements between rows
  bool reused = false;             // THX_REUSED
  const char *lo = nullptr, *hi = nullptr;  // the bytes it spans, for the overlap check
};

// Takes `a` apart into rows: the last `trailing` (0 or 1) axes are the columns, the axes before them have to collapse
// to one stride.  `dtype` < 0: any (the caller looks at it).  Columns have to lie side by side (THX_ERR_UNSUPPORTED
// otherwise, as for rows at more than one stride).
inline int rows_of(const char* what, const char* name, const thx_array* a, int dtype, int trailing, int flags, Rows* r) {
  if (!a) return fail(THX_ERR_ARG, "%s: %s is missing", what, name);
  if (a->nd < trailing || a->nd > THX_MAX_ND)
    return fail(THX_ERR_TYPE, "%s: %s has rank %d", what, name, a->nd);
  if (a->dtype & (THX_HOST_SCALAR | THX_INDEX))
    return fail(THX_ERR_TYPE, "%s: %s must be a device array", what, name);
  r->dtype = a->dtype & ~THX_REUSED;
  r->reused = (a->dtype & THX_REUSED) != 0;
  const int isz = dtype_size(r->dtype);
  if (!isz || (dtype >= 0 && r->dtype != dtype))
    return fail(THX_ERR_TYPE, "%s: %s has dtype code %d, expected %d", what, name, r->dtype, dtype);
  if (null_base(*a, (flags & THX_DRY_RUN) != 0)) return fail(THX_ERR_ARG, "%s: %s has no base address", what, name);
  r->nd = a->nd;
  r->ptr = (char*)a->base + a->offset_bytes;
  if ((uintptr_t)r->ptr % isz) return fail(THX_ERR_TYPE, "%s: %s is not aligned to its element size", what, name);
  const int lead = a->nd - trailing;
  r->lo = r->hi = r->ptr;
  bool empty = false;
  for (int d = 0; d < a->nd; ++d) {
    if (a->shape[d] < 0) return fail(THX_ERR_ARG, "%s: %s has a negative extent", what, name);
    if (a->shape[d] > 1 && a->strides_bytes[d] % isz)
      return fail(THX_ERR_TYPE, "%s: a stride of %s is not a multiple of its element size", what, name);
    if (a->shape[d] == 0) empty = true;
  }
  r->cols = trailing ? a->shape[lead] : 1;
  r->rows = 1;
  for (int d = 0; d < lead; ++d) r->rows *= a->shape[d];
  if (empty) {
    r->stride = r->cols;
    return THX_OK;
  }
  if (trailing && r->cols > 1 && a->strides_bytes[lead] != isz)
    return fail(THX_ERR_UNSUPPORTED, "%s: the columns of %s do not lie side by side", what, name);
  // from the innermost axis out: an axis of more than one element continues the rows where the ones inside it end
  int64_t stride = 0, span = 0;
  bool first = true;
  for (int d = lead - 1; d >= 0; --d) {
    if (a->shape[d] == 1) continue;
    if (first) {
      stride = a->strides_bytes[d];
      span = stride * a->shape[d];
      first = false;
    } else {
      if (a->strides_bytes[d] != span)
        return fail(THX_ERR_UNSUPPORTED, "%s: the rows of %s do not lie at one stride", what, name);
      span *= a->shape[d];
    }
  }
  r->stride = first ? r->cols : stride / isz;
  const int64_t reach = (r->rows - 1) * r->stride * isz, width = r->cols * isz;
  r->lo = r->ptr + std::min<int64_t>(reach, 0);
  r->hi = r->ptr + std::max<int64_t>(reach, 0) + width;
  return THX_OK;
}

// An operand of the shape of the leading axes of `x` (one value per row), or of those and `cols` columns.
inline int like_rows(const char* what, const char* name, const thx_array* a, const thx_array* x, int dtype, int64_t cols,
                     int flags, Rows* r) {
  int rc = rows_of(what, name, a, dtype, cols >= 0 ? 1 : 0, flags, r);
  if (rc) return rc;
  const int lead = x->nd - 1;
  bool same = a->nd == lead + (cols >= 0 ? 1 : 0) && (cols < 0 || a->shape[lead] == cols);
  for (int d = 0; same && d < lead; ++d) same = a->shape[d] == x->shape[d];
  if (!same) return fail(THX_ERR_SHAPE, "Input dimension mis-match. (%s: %s does not have the rows of the input)", what, name);
  return THX_OK;
}

inline int contiguous_rows(const char* what, const char* name, const Rows& r) {
  if (r.rows > 1 && r.stride != r.cols) return fail(THX_ERR_TYPE, "%s: %s must be C-contiguous", what, name);
  return THX_OK;
}

// The kernels read operands again after they have begun to write: a result must not lie over one.
inline int no_overlap(const char* what, const Rows* outs, int n_out, const Rows* ins, int n_in) {
  for (int o = 0; o < n_out; ++o) {
    for (int i = 0; i < n_in; ++i)
      if (outs[o].lo < ins[i].hi && ins[i].lo < outs[o].hi)
        return fail(THX_ERR_ARG, "%s: a result overlaps an operand", what);
    for (int p = 0; p < o; ++p)
      if (outs[o].lo < outs[p].hi && outs[p].lo < outs[o].hi)
        return fail(THX_ERR_ARG, "%s: two results overlap", what);
  }
  return THX_OK;
}

inline int check_workspace(const char* what, void* ws, size_t have, size_t need, int flags) {
  if (need && have < need) return fail(THX_ERR_ARG, "%s: needs a workspace of %zu bytes, got %zu", what, need, have);
  if (need && !ws && !(flags & THX_DRY_RUN)) return fail(THX_ERR_ARG, "%s: the workspace has no address", what);
  if ((uintptr_t)ws % 16) return fail(THX_ERR_ARG, "%s: the workspace must be aligned to 16 bytes", what);
  return THX_OK;
}

// Whether a result as large as the rows `x` it comes from is written past the caches: where the two together exceed what
// the last-level cache holds for a reader, unless the caller says that one follows.  Measured on gradients of 2048 rows
// of 32000 floats 138 -> 125 us, of 4096 rows of 128000 halves 579 -> 555; below the border such stores are slower.
inline bool stream_out(const Rows& x, const Rows& out) {
  return !out.reused && nt_streaming(2 * x.rows * x.cols * dtype_size(x.dtype));
}

inline int compute_units() { return rt().cus ? rt().cus : 256; }

}  // namespace thx
