// Host side of the sequence operators (include/nsfps.h, "Sequence
// operators"): argument checks and launches.  The calls share nothing: no
// lock, no workspace of the library's own, no wait.
#include "nsfps_sequence.h"
#include "nsfps_status.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <utility>

namespace nsfps {
namespace {

constexpr uint64_t kMaxCount = 0x7fffffffull;
constexpr uint64_t kMaxElems = 1ull << 46;  // offsets stay far inside 64 bits

nsfps_status need_device() {
  static std::atomic<bool> seen{false};  // devices do not go away
  if (seen.load(std::memory_order_relaxed)) return NSFPS_OK;
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n <= 0)
    return fail(NSFPS_EDEVICE, "no HIP device available (nsfps has no CPU path)");
  seen.store(true, std::memory_order_relaxed);
  return NSFPS_OK;
}

bool is_dtype(uint32_t t) { return t == NSFPS_F32 || t == NSFPS_BF16; }
uint64_t size_of(uint32_t t) { return t == NSFPS_F32 ? 4 : 2; }

nsfps_status check_pointer(const void *p, uint64_t align, const char *what) {
  if (!p) return fail(NSFPS_EINVAL, "null pointer: %s", what);
  if ((uintptr_t)p % align)
    return fail(NSFPS_EINVAL, "%s is not aligned to %d bytes", what, (int)align);
  return NSFPS_OK;
}
// a pointer that may be null
nsfps_status check_optional(const void *p, uint64_t align, const char *what) {
  return p ? check_pointer(p, align, what) : NSFPS_OK;
}

#define TRY(expr)                        \
  do {                                   \
    const nsfps_status rc_ = (expr);     \
    if (rc_ != NSFPS_OK) return rc_;     \
  } while (0)

// Rows of `width` elements that lie apart: a batch may be interleaved with
// the length either way round.
nsfps_status check_rows(const nsfps_rows &r, uint64_t batch, uint64_t length, uint64_t width,
                        uint32_t dtype, bool written, const char *what) {
  TRY(check_pointer(r.p, size_of(dtype), what));
  if (r.row_stride > kMaxElems || r.batch_stride > kMaxElems ||
      (batch && r.batch_stride > kMaxElems / batch) ||
      (length && r.row_stride > kMaxElems / length))
    return fail(NSFPS_EINVAL, "strides of %s are too large", what);
  if (!written) return NSFPS_OK;  // inputs may repeat rows (a stride of 0)
  const bool rows_apart = length <= 1 || r.row_stride >= width;
  const uint64_t row_span = (length - 1) * r.row_stride + width;
  const uint64_t batch_span = (batch - 1) * r.batch_stride + width;
  const bool batches_apart = batch <= 1 || r.batch_stride >= row_span ||
                             (r.batch_stride >= width && (length <= 1 || r.row_stride >= batch_span));
  if (!rows_apart || !batches_apart)
    return fail(NSFPS_EINVAL, "rows of %s overlap: %llu elements, batch stride %llu, row stride %llu",
                what, (unsigned long long)width, (unsigned long long)r.batch_stride,
                (unsigned long long)r.row_stride);
  return NSFPS_OK;
}

// Whether two tensors of these sizes share an element, as far as their strides
// tell: the same first element, or the same strides.  `out` keeps its rows apart
// (check_rows), so the offsets of two rows of it that can meet are the few
// nearest to the tensors' distance.
bool rows_meet(const nsfps_rows &out, uint64_t out_width, const nsfps_rows &in, uint64_t in_width,
               uint64_t batch, uint64_t length, uint32_t dtype) {
  if (out.p == in.p) return true;
  if ((batch > 1 && out.batch_stride != in.batch_stride) ||
      (length > 1 && out.row_stride != in.row_stride))
    return false;
  struct Step {
    int64_t stride, most;  // elements; how often it may be taken either way
  } far{(int64_t)out.batch_stride, (int64_t)batch - 1},
      near{(int64_t)out.row_stride, (int64_t)length - 1};
  if (near.most && (!far.most || near.stride > far.stride)) std::swap(far, near);
  const int64_t d = ((intptr_t)in.p - (intptr_t)out.p) / (int64_t)size_of(dtype),
                span = far.most * far.stride + near.most * near.stride;
  if (d >= span + (int64_t)out_width || -d >= span + (int64_t)in_width) return false;
  const auto nearest = [](const Step &s, int64_t at, int64_t k) {  // at, some steps back
    const int64_t q = s.most ? std::max(-s.most, std::min(s.most, at / s.stride + k)) : 0;
    return at - q * s.stride;
  };
  for (int64_t k = -1; k <= 1; ++k)
    for (int64_t j = -1; j <= 1; ++j) {
      const int64_t left = nearest(near, nearest(far, d, k), j);
      if (left < (int64_t)out_width && -left < (int64_t)in_width) return true;
    }
  return false;
}

nsfps_status check_apart(const nsfps_rows &out, const nsfps_rows &in, const nsfps_conv_args &a,
                         const char *what) {
  if (rows_meet(out, a.channels, in, a.channels, a.batch, a.length, a.dtype))
    return fail(NSFPS_EINVAL, "%s overlap: tokens beside a row are read after it is written", what);
  return NSFPS_OK;
}

// Rows of one tensor of an operator whose lanes take their values before they write
// the same places: an output may be its own input's very rows (check_own), and must
// share nothing with another tensor's (check_other).
struct Tensor {
  nsfps_rows rows;
  uint64_t width;
  const char *what;
};
struct Sizes {
  uint64_t batch, length;
  uint32_t dtype;
};
nsfps_status check_other(const Tensor &out, const Tensor &in, const Sizes &n) {
  if (!out.width || !in.width) return NSFPS_OK;  // no heads
  const auto whole = [&](const Tensor &t) {  // one piece of memory
    return (n.length == 1 || t.rows.row_stride == t.width) &&
           (n.batch == 1 || t.rows.batch_stride == n.length * t.width);
  };
  const uint64_t bytes = n.batch * n.length * size_of(n.dtype), o = (uintptr_t)out.rows.p,
                 i = (uintptr_t)in.rows.p;
  const bool meet = whole(out) && whole(in)
                        ? o < i + bytes * in.width && i < o + bytes * out.width
                        : rows_meet(out.rows, out.width, in.rows, in.width, n.batch, n.length, n.dtype);
  if (meet)
    return fail(NSFPS_EINVAL, "%s and %s overlap", out.what, in.what);
  return NSFPS_OK;
}
nsfps_status check_own(const Tensor &out, const Tensor &in, const Sizes &n) {
  const bool same = out.rows.p == in.rows.p &&
                    (n.batch <= 1 || out.rows.batch_stride == in.rows.batch_stride) &&
                    (n.length <= 1 || out.rows.row_stride == in.rows.row_stride);
  return same ? NSFPS_OK : check_other(out, in, n);
}

// Rows of a matrix, in bytes.
struct Span {
  const void *p;
  uint64_t rows, stride, width;
  const char *what;
};
// Whether they share a byte, as far as their strides tell: exactly where one of the two
// has no gaps, or where both have the same stride.
bool spans_meet(const Span &a, const Span &b) {
  if (!a.rows || !b.rows) return false;
  if (a.p == b.p) return true;
  const bool a_whole = a.rows == 1 || a.stride == a.width, b_whole = b.rows == 1 || b.stride == b.width;
  const auto last = [](const Span &s) { return (int64_t)((s.rows - 1) * s.stride + s.width); };
  const int64_t d = (intptr_t)b.p - (intptr_t)a.p;  // from a's first to b's first
  if (d >= last(a) || -d >= last(b)) return false;
  // a whole one, from `from` to `to` in the other's bytes, meets the first row that ends
  // behind `from`
  const auto meets = [](const Span &s, int64_t from, int64_t to) {
    const int64_t w = (int64_t)s.width, st = (int64_t)std::max<uint64_t>(s.stride, 1);
    const int64_t row = from < w ? 0 : (from - w) / st + 1;
    return row < (int64_t)s.rows && row * (int64_t)s.stride < to;
  };
  if (a_whole) return meets(b, -d, last(a) - d);
  if (b_whole) return meets(a, d, d + last(b));
  if (a.stride != b.stride) return false;
  const int64_t st = (int64_t)a.stride, in = (d % st + st) % st;  // b's row in a's period
  return in < (int64_t)a.width || in + (int64_t)b.width > st;
}
nsfps_status check_spans(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  for (auto out = outs.begin(); out != outs.end(); ++out) {
    for (auto other = outs.begin(); other != out; ++other)
      if (spans_meet(*out, *other))
        return fail(NSFPS_EINVAL, "%s and %s overlap", other->what, out->what);
    for (const Span &in : ins)
      if (spans_meet(*out, in)) return fail(NSFPS_EINVAL, "%s and %s overlap", out->what, in.what);
  }
  return NSFPS_OK;
}

nsfps_status check_workspace(const void *p, uint64_t have, uint64_t need) {
  if (!need) return NSFPS_OK;
  TRY(check_pointer(p, 256, "workspace"));
  if (have < need)
    return fail(NSFPS_EINVAL, "workspace of %llu bytes: %llu are needed",
                (unsigned long long)have, (unsigned long long)need);
  return NSFPS_OK;
}

// ------------------------------------------------------------- embedding

nsfps_status check_embed_sizes(const nsfps_embed_args *a, bool grad) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  if (!is_dtype(a->dtype) || (grad && !is_dtype(a->grad_dtype)))
    return fail(NSFPS_EINVAL, "unknown type");
  if (a->width == 0) return fail(NSFPS_EINVAL, "width must be >= 1");
  if (a->tokens > kMaxCount || a->rows > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^31-1 tokens or rows");
  if (a->width > 65536) return fail(NSFPS_EUNSUPPORTED, "width above 65536");
  return NSFPS_OK;
}

nsfps_status check_embed(const nsfps_embed_args *a, bool grad) {
  TRY(check_embed_sizes(a, grad));
  if ((a->rows && a->table_stride < a->width) || (a->tokens && a->out_stride < a->width))
    return fail(NSFPS_EINVAL, "strides must be >= width");
  if (a->table_stride > kMaxElems / (a->rows + 1) || a->out_stride > kMaxElems / (a->tokens + 1))
    return fail(NSFPS_EINVAL, "strides are too large");
  if (a->rows) TRY(check_pointer(a->d_table, size_of(grad ? a->grad_dtype : a->dtype), "d_table"));
  if (a->tokens) {
    TRY(check_pointer(a->d_tokens, 4, "d_tokens"));
    TRY(check_pointer(a->d_out, size_of(a->dtype), "d_out"));
  }
  return NSFPS_OK;
}

// ----------------------------------------------------------- convolution

nsfps_status check_conv_sizes(const nsfps_conv_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  if (!is_dtype(a->dtype)) return fail(NSFPS_EINVAL, "unknown type");
  if (a->channels == 0) return fail(NSFPS_EINVAL, "channels must be >= 1");
  if (a->width < 2 || a->width > 4)
    return fail(NSFPS_EUNSUPPORTED, "width %u: 2 to 4 are supported", a->width);
  if (a->channels > 1u << 24) return fail(NSFPS_EUNSUPPORTED, "more than 2^24 channels");
  if (a->batch > kMaxCount || a->length > kMaxCount || a->batch * a->length > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^31-1 tokens");
  return NSFPS_OK;
}

nsfps_status check_conv(const nsfps_conv_args *a, bool grad) {
  TRY(check_conv_sizes(a));
  if (a->batch && a->length) {
    TRY(check_rows(a->x, a->batch, a->length, a->channels, a->dtype, false, "x"));
    if (!grad) TRY(check_rows(a->y, a->batch, a->length, a->channels, a->dtype, true, "y"));
  }
  TRY(check_pointer(a->d_weight, size_of(a->dtype), "d_weight"));
  TRY(check_optional(a->d_bias, size_of(a->dtype), "d_bias"));
  TRY(check_optional(a->d_lengths, 4, "d_lengths"));
  TRY(check_optional(a->d_positions, 4, "d_positions"));
  TRY(check_optional(a->d_slots, 4, "d_slots"));
  TRY(check_optional(a->d_cache, size_of(a->dtype), "d_cache"));
  if (grad && (a->d_positions || a->d_slots || a->d_cache))
    return fail(NSFPS_EINVAL, "the gradient starts every sequence anew: no positions, no cache");
  if (!grad && a->d_positions && !a->d_cache)
    return fail(NSFPS_EINVAL, "positions continue from a cache, and d_cache is null");
  return NSFPS_OK;
}

// ------------------------------------------------------------------ scan

nsfps_status check_heads(uint64_t batch, uint32_t heads, uint32_t groups, uint32_t head_dim,
                         uint32_t state_dim, uint32_t dtype) {
  if (!is_dtype(dtype)) return fail(NSFPS_EINVAL, "unknown type");
  if (heads == 0 || groups == 0 || head_dim == 0 || state_dim == 0)
    return fail(NSFPS_EINVAL, "heads, groups, head_dim and state_dim must be >= 1");
  if (heads % groups) return fail(NSFPS_EINVAL, "%u groups do not divide %u heads", groups, heads);
  if (head_dim > 128 || state_dim > 128)
    return fail(NSFPS_EUNSUPPORTED, "head_dim %u, state_dim %u: at most 128 are supported", head_dim,
                state_dim);
  if (heads > 1u << 20 || batch > (1ull << 20) / heads)
    return fail(NSFPS_EUNSUPPORTED, "batch * heads above 2^20");
  return NSFPS_OK;
}

nsfps_status check_scan_sizes(const nsfps_scan_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  TRY(check_heads(a->batch, a->heads, a->groups, a->head_dim, a->state_dim, a->dtype));
  if (a->length > kMaxCount || a->batch * a->length > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^31-1 tokens");
  return NSFPS_OK;
}

nsfps_status check_scan(const nsfps_scan_args *a, bool grad) {
  TRY(check_scan_sizes(a));
  if (a->batch && a->length) {
    const uint64_t hp = (uint64_t)a->heads * a->head_dim, gn = (uint64_t)a->groups * a->state_dim;
    TRY(check_rows(a->x, a->batch, a->length, hp, a->dtype, false, "x"));
    TRY(check_rows(a->b, a->batch, a->length, gn, a->dtype, false, "b"));
    TRY(check_rows(a->c, a->batch, a->length, gn, a->dtype, false, "c"));
    TRY(check_rows(a->dt, a->batch, a->length, a->heads, a->dtype, false, "dt"));
    if (!grad) TRY(check_rows(a->y, a->batch, a->length, hp, a->dtype, true, "y"));
  }
  TRY(check_pointer(a->d_a, 4, "d_a"));
  TRY(check_optional(a->d_d, 4, "d_d"));
  TRY(check_optional(a->d_dt_bias, 4, "d_dt_bias"));
  TRY(check_optional(a->d_lengths, 4, "d_lengths"));
  TRY(check_optional(a->d_positions, 4, "d_positions"));
  TRY(check_optional(a->d_slots, 4, "d_slots"));
  TRY(check_optional(a->d_state, 4, "d_state"));
  if (grad && (a->d_positions || a->d_slots || a->d_state))
    return fail(NSFPS_EINVAL, "the gradient starts every sequence anew: no positions, no state");
  if (!grad && a->d_positions && !a->d_state)
    return fail(NSFPS_EINVAL, "positions continue from a state, and d_state is null");
  return NSFPS_OK;
}

nsfps_status check_step(const nsfps_step_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  TRY(check_heads(a->batch, a->heads, a->groups, a->head_dim, a->state_dim, a->dtype));
  if (a->width < 2 || a->width > 4)
    return fail(NSFPS_EUNSUPPORTED, "width %u: 2 to 4 are supported", a->width);
  if (!a->batch) return NSFPS_OK;
  const uint64_t hp = (uint64_t)a->heads * a->head_dim,
                 ch = hp + 2ull * a->groups * a->state_dim, z = size_of(a->dtype);
  if (a->batch > 1 && a->y_stride < hp) return fail(NSFPS_EINVAL, "rows of y overlap");
  if (a->xbc_stride > kMaxElems / a->batch || a->dt_stride > kMaxElems / a->batch ||
      a->y_stride > kMaxElems / a->batch)
    return fail(NSFPS_EINVAL, "strides are too large");
  if (ch > 1u << 24) return fail(NSFPS_EUNSUPPORTED, "more than 2^24 channels");
  TRY(check_pointer(a->d_xbc, z, "d_xbc"));
  TRY(check_pointer(a->d_weight, z, "d_weight"));
  TRY(check_optional(a->d_bias, z, "d_bias"));
  TRY(check_pointer(a->d_dt, z, "d_dt"));
  TRY(check_pointer(a->d_a, 4, "d_a"));
  TRY(check_optional(a->d_d, 4, "d_d"));
  TRY(check_optional(a->d_dt_bias, 4, "d_dt_bias"));
  TRY(check_pointer(a->d_positions, 4, "d_positions"));
  TRY(check_optional(a->d_slots, 4, "d_slots"));
  TRY(check_pointer(a->d_cache, z, "d_cache"));
  TRY(check_pointer(a->d_state, 4, "d_state"));
  TRY(check_pointer(a->d_y, z, "d_y"));
  return NSFPS_OK;
}

// ------------------------------------------------------------------ norms

nsfps_status check_norm_sizes(const nsfps_norm_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  if (!is_dtype(a->dtype)) return fail(NSFPS_EINVAL, "unknown type");
  if (a->head_dim == 0 || (a->q_heads == 0 && a->k_heads == 0))
    return fail(NSFPS_EINVAL, "head_dim and one of q_heads and k_heads must be >= 1");
  if (a->head_dim > 256)
    return fail(NSFPS_EUNSUPPORTED, "head_dim %u: at most 256 is supported", a->head_dim);
  if (a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return fail(NSFPS_EINVAL, "rotary_dim %u must be even and at most head_dim %u", a->rotary_dim,
                a->head_dim);
  if (!(a->eps > 0.f) || !std::isfinite(a->eps))
    return fail(NSFPS_EINVAL, "eps must be finite and above 0");
  if (((uint64_t)a->q_heads + a->k_heads) * a->head_dim > 1u << 24)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^24 channels");
  if (a->batch > kMaxCount || a->length > kMaxCount || a->batch * a->length > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^31-1 tokens");
  return NSFPS_OK;
}

// Outputs (y, or dx) of queries and keys: over their own inputs or gradients, or apart.
nsfps_status check_norm_places(const nsfps_norm_args &a, const nsfps_rows &q_out,
                               const nsfps_rows &k_out, const nsfps_norm_grads *g) {
  const uint64_t d = a.head_dim, qw = a.q_heads * d, kw = a.k_heads * d;
  const Sizes n = {a.batch, a.length, a.dtype};
  const Tensor q = {a.q, qw, "q"}, k = {a.k, kw, "k"}, qo = {q_out, qw, g ? "dq" : "q_out"},
               ko = {k_out, kw, g ? "dk" : "k_out"};
  TRY(check_other(qo, ko, n));
  TRY(check_own(qo, q, n));
  TRY(check_own(ko, k, n));
  TRY(check_other(qo, k, n));
  TRY(check_other(ko, q, n));
  if (!g) return NSFPS_OK;
  const Tensor dq = {g->dq_out, qw, "dq_out"}, dk = {g->dk_out, kw, "dk_out"};
  TRY(check_own(qo, dq, n));
  TRY(check_own(ko, dk, n));
  TRY(check_other(qo, dk, n));
  return check_other(ko, dq, n);
}

nsfps_status check_norm(const nsfps_norm_args *a, bool grad) {
  TRY(check_norm_sizes(a));
  if (a->batch && a->length) {
    const uint64_t b = a->batch, l = a->length, d = a->head_dim;
    if (a->q_heads) {
      TRY(check_rows(a->q, b, l, a->q_heads * d, a->dtype, false, "q"));
      if (!grad) TRY(check_rows(a->q_out, b, l, a->q_heads * d, a->dtype, true, "q_out"));
    }
    if (a->k_heads) {
      TRY(check_rows(a->k, b, l, a->k_heads * d, a->dtype, false, "k"));
      if (!grad) TRY(check_rows(a->k_out, b, l, a->k_heads * d, a->dtype, true, "k_out"));
    }
  }
  TRY(check_optional(a->d_q_weight, size_of(a->dtype), "d_q_weight"));
  TRY(check_optional(a->d_k_weight, size_of(a->dtype), "d_k_weight"));
  if (a->rotary_dim) TRY(check_pointer(a->d_freq, 4, "d_freq"));
  TRY(check_optional(a->d_lengths, 4, "d_lengths"));
  TRY(check_optional(a->d_positions, 4, "d_positions"));
  return NSFPS_OK;
}

// ---------------------------------------------------------------- dropout

nsfps_status check_dropout(const nsfps_dropout_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  if (!is_dtype(a->dtype)) return fail(NSFPS_EINVAL, "unknown type");
  if (a->channels == 0) return fail(NSFPS_EINVAL, "channels must be >= 1");
  if (a->channels > 1u << 24) return fail(NSFPS_EUNSUPPORTED, "more than 2^24 channels");
  if (!(a->p >= 0.f && a->p <= 1.f)) return fail(NSFPS_EINVAL, "p must be between 0 and 1");
  if (a->batch > kMaxCount || a->length > kMaxCount || a->batch * a->length > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^31-1 tokens");
  if (a->batch && a->length) {
    TRY(check_rows(a->x, a->batch, a->length, a->channels, a->dtype, false, "x"));
    if (a->residual.p)
      TRY(check_rows(a->residual, a->batch, a->length, a->channels, a->dtype, false, "residual"));
    TRY(check_rows(a->y, a->batch, a->length, a->channels, a->dtype, true, "y"));
    const Sizes n = {a->batch, a->length, a->dtype};
    const Tensor y = {a->y, a->channels, "y"};
    TRY(check_own(y, {a->x, a->channels, "x"}, n));
    if (a->residual.p) TRY(check_own(y, {a->residual, a->channels, "residual"}, n));
  }
  TRY(check_pointer(a->d_seed, 8, "d_seed"));
  TRY(check_optional(a->d_lengths, 4, "d_lengths"));
  return NSFPS_OK;
}

// ------------------------------------------------------- vocabulary loss

nsfps_status check_loss_sizes(const nsfps_loss_args *a) {
  if (!a) return fail(NSFPS_EINVAL, "null pointer: args");
  if (!is_dtype(a->dtype)) return fail(NSFPS_EINVAL, "unknown type");
  if (a->width == 0) return fail(NSFPS_EINVAL, "width must be >= 1");
  if (a->tokens > 1u << 30 || a->rows > kMaxCount)
    return fail(NSFPS_EUNSUPPORTED, "more than 2^30 tokens or 2^31-1 rows");
  if (a->width > 65536) return fail(NSFPS_EUNSUPPORTED, "width above 65536");
  return NSFPS_OK;
}

nsfps_status check_row_stride(uint64_t stride, uint64_t rows, uint64_t width, const char *what) {
  if (rows && stride < width) return fail(NSFPS_EINVAL, "%s must be >= width", what);
  if (stride > kMaxElems / (rows + 1)) return fail(NSFPS_EINVAL, "%s is too large", what);
  return NSFPS_OK;
}

nsfps_status check_loss(const nsfps_loss_args *a, bool grad) {
  TRY(check_loss_sizes(a));
  // (logits are found in powers of two)
  if (!std::isfinite(a->scale) || !std::isfinite(a->scale * 1.44269504f))
    return fail(NSFPS_EINVAL, "scale and scale * log2(e) must be finite");
  TRY(check_row_stride(a->x_stride, a->tokens, a->width, "x_stride"));
  TRY(check_row_stride(a->table_stride, a->rows, a->width, "table_stride"));
  if (a->rows) TRY(check_pointer(a->d_table, size_of(a->dtype), "d_table"));
  if (a->tokens) {
    TRY(check_pointer(a->d_x, size_of(a->dtype), "d_x"));
    TRY(check_pointer(a->d_targets, 4, "d_targets"));
    if (!grad) TRY(check_pointer(a->d_loss, 4, "d_loss"));
    TRY(check_pointer(a->d_lse, 4, "d_lse"));
  }
  return NSFPS_OK;
}

// The loss writes rows while others are still to be read: nothing may overlap.
struct LossSpans {
  Span x, table, targets, lse;
};
LossSpans loss_spans(const nsfps_loss_args &a) {
  const uint64_t z = size_of(a.dtype), n = a.tokens;
  return {{a.d_x, n, a.x_stride * z, a.width * z, "d_x"},
          {a.d_table, a.rows, a.table_stride * z, a.width * z, "d_table"},
          {a.d_targets, n, 4, 4, "d_targets"},
          {a.d_lse, n, 4, 4, "d_lse"}};
}

nsfps_status check_loss_grads(const nsfps_loss_grads *g) {
  if (!g) return fail(NSFPS_EINVAL, "null pointer: grads");
  if (!is_dtype(g->grad_dtype)) return fail(NSFPS_EINVAL, "unknown type");
  return NSFPS_OK;
}

}  // namespace
}  // namespace nsfps

using namespace nsfps;

extern "C" {

nsfps_status nsfps_init_sequence_device(void) {
  return guarded([&]() -> nsfps_status {
    TRY(need_device());
    HIP_TRY(preload_embed_kernels());
    HIP_TRY(preload_conv_kernels());
    HIP_TRY(preload_scan_kernels());
    HIP_TRY(preload_scan_grad_kernels());
    HIP_TRY(preload_norm_kernels());
    HIP_TRY(preload_dropout_kernels());
    HIP_TRY(preload_loss_kernels());
    return NSFPS_OK;
  });
}

nsfps_status nsfps_embed_device(const nsfps_embed_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_embed(args, false));
    if (!args->tokens) return NSFPS_OK;
    TRY(need_device());
    HIP_TRY(launch_embed(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_embed_grad_workspace_bytes(const nsfps_embed_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_embed_sizes(args, true));
    *bytes = embed_grad_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_embed_grad_device(const nsfps_embed_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_embed(args, true));
    if (!args->rows) return NSFPS_OK;
    TRY(check_workspace(args->workspace, args->workspace_bytes, embed_grad_bytes(*args)));
    TRY(need_device());
    HIP_TRY(launch_embed_grad(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_conv_device(const nsfps_conv_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_conv(args, false));
    if (!args->batch || !args->length) return NSFPS_OK;
    TRY(check_apart(args->y, args->x, *args, "x and y"));
    TRY(need_device());
    HIP_TRY(launch_conv(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_conv_grad_workspace_bytes(const nsfps_conv_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_conv_sizes(args));
    *bytes = conv_grad_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_conv_grad_device(const nsfps_conv_args *args, const nsfps_conv_grads *grads,
                                    void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_conv(args, true));
    if (!grads) return fail(NSFPS_EINVAL, "null pointer: grads");
    if (args->batch && args->length) {
      TRY(check_rows(grads->dy, args->batch, args->length, args->channels, args->dtype, false, "dy"));
      TRY(check_rows(grads->dx, args->batch, args->length, args->channels, args->dtype, true, "dx"));
    }
    TRY(check_pointer(grads->d_dweight, 4, "d_dweight"));
    TRY(check_optional(grads->d_dbias, 4, "d_dbias"));
    TRY(check_workspace(args->workspace, args->workspace_bytes, conv_grad_bytes(*args)));
    if (args->batch && args->length) {
      TRY(check_apart(grads->dx, args->x, *args, "x and dx"));
      TRY(check_apart(grads->dx, grads->dy, *args, "dy and dx"));
    }
    TRY(need_device());
    HIP_TRY(launch_conv_grad(*args, *grads, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_scan_workspace_bytes(const nsfps_scan_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_scan_sizes(args));
    *bytes = scan_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_scan_device(const nsfps_scan_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_scan(args, false));
    if (!args->batch || !args->length) return NSFPS_OK;
    TRY(check_workspace(args->workspace, args->workspace_bytes, scan_bytes(*args)));
    TRY(need_device());
    HIP_TRY(launch_scan(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_scan_grad_workspace_bytes(const nsfps_scan_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_scan_sizes(args));
    *bytes = scan_grad_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_scan_grad_device(const nsfps_scan_args *args, const nsfps_scan_grads *grads,
                                    void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_scan(args, true));
    if (!grads) return fail(NSFPS_EINVAL, "null pointer: grads");
    if (args->batch && args->length) {
      const uint64_t hp = (uint64_t)args->heads * args->head_dim,
                     gn = (uint64_t)args->groups * args->state_dim, b = args->batch,
                     l = args->length;
      const uint32_t t = args->dtype;
      TRY(check_rows(grads->dy, b, l, hp, t, false, "dy"));
      TRY(check_rows(grads->dx, b, l, hp, t, true, "dx"));
      TRY(check_rows(grads->db, b, l, gn, t, true, "db"));
      TRY(check_rows(grads->dc, b, l, gn, t, true, "dc"));
      TRY(check_rows(grads->ddt, b, l, args->heads, t, true, "ddt"));
    }
    TRY(check_pointer(grads->d_da, 4, "d_da"));
    TRY(check_optional(grads->d_dd, 4, "d_dd"));
    TRY(check_optional(grads->d_ddt_bias, 4, "d_ddt_bias"));
    TRY(check_workspace(args->workspace, args->workspace_bytes, scan_grad_bytes(*args)));
    TRY(need_device());
    HIP_TRY(launch_scan_grad(*args, *grads, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_scan_step_device(const nsfps_step_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_step(args));
    if (!args->batch) return NSFPS_OK;
    TRY(need_device());
    HIP_TRY(launch_scan_step(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_norm_device(const nsfps_norm_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_norm(args, false));
    if (!args->batch || !args->length) return NSFPS_OK;
    TRY(check_norm_places(*args, args->q_out, args->k_out, nullptr));
    TRY(need_device());
    HIP_TRY(launch_norm(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_norm_grad_workspace_bytes(const nsfps_norm_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_norm_sizes(args));
    *bytes = norm_grad_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_norm_grad_device(const nsfps_norm_args *args, const nsfps_norm_grads *grads,
                                    void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_norm(args, true));
    if (!grads) return fail(NSFPS_EINVAL, "null pointer: grads");
    if (args->batch && args->length) {
      const uint64_t b = args->batch, l = args->length, d = args->head_dim;
      const uint32_t t = args->dtype;
      if (args->q_heads) {
        TRY(check_rows(grads->dq_out, b, l, args->q_heads * d, t, false, "dq_out"));
        TRY(check_rows(grads->dq, b, l, args->q_heads * d, t, true, "dq"));
      }
      if (args->k_heads) {
        TRY(check_rows(grads->dk_out, b, l, args->k_heads * d, t, false, "dk_out"));
        TRY(check_rows(grads->dk, b, l, args->k_heads * d, t, true, "dk"));
      }
      TRY(check_norm_places(*args, grads->dq, grads->dk, grads));
    }
    TRY(check_optional(grads->d_dq_weight, 4, "d_dq_weight"));
    TRY(check_optional(grads->d_dk_weight, 4, "d_dk_weight"));
    TRY(check_workspace(args->workspace, args->workspace_bytes, norm_grad_bytes(*args)));
    TRY(need_device());
    HIP_TRY(launch_norm_grad(*args, *grads, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_dropout_device(const nsfps_dropout_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_dropout(args));
    if (!args->batch || !args->length) return NSFPS_OK;
    TRY(need_device());
    HIP_TRY(launch_dropout(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_loss_workspace_bytes(const nsfps_loss_args *args, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_loss_sizes(args));
    *bytes = loss_bytes(*args);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_loss_device(const nsfps_loss_args *args, void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_loss(args, false));
    if (!args->tokens) return NSFPS_OK;
    const LossSpans s = loss_spans(*args);
    TRY(check_spans({s.lse, {args->d_loss, args->tokens, 4, 4, "d_loss"}}, {s.x, s.table, s.targets}));
    TRY(check_workspace(args->workspace, args->workspace_bytes, loss_bytes(*args)));
    TRY(need_device());
    HIP_TRY(launch_loss(*args, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

nsfps_status nsfps_loss_grad_workspace_bytes(const nsfps_loss_args *args,
                                             const nsfps_loss_grads *grads, uint64_t *bytes) {
  return guarded([&]() -> nsfps_status {
    if (!bytes) return fail(NSFPS_EINVAL, "null pointer: bytes");
    TRY(check_loss_sizes(args));
    TRY(check_loss_grads(grads));
    *bytes = loss_grad_bytes(*args, *grads);
    return NSFPS_OK;
  });
}

nsfps_status nsfps_loss_grad_device(const nsfps_loss_args *args, const nsfps_loss_grads *grads,
                                    void *stream) {
  return guarded([&]() -> nsfps_status {
    TRY(check_loss(args, true));
    TRY(check_loss_grads(grads));
    TRY(check_row_stride(grads->dx_stride, args->tokens, args->width, "dx_stride"));
    TRY(check_row_stride(grads->dtable_stride, args->rows, args->width, "dtable_stride"));
    if (args->tokens) {
      TRY(check_pointer(grads->d_dloss, 4, "d_dloss"));
      TRY(check_pointer(grads->d_dx, size_of(args->dtype), "d_dx"));
    }
    if (args->rows) TRY(check_pointer(grads->d_dtable, size_of(grads->grad_dtype), "d_dtable"));
    if (!args->tokens && !args->rows) return NSFPS_OK;
    const LossSpans s = loss_spans(*args);
    const uint64_t z = size_of(args->dtype), gz = size_of(grads->grad_dtype), w = args->width;
    TRY(check_spans({{grads->d_dx, args->tokens, grads->dx_stride * z, w * z, "d_dx"},
                     {grads->d_dtable, args->rows, grads->dtable_stride * gz, w * gz, "d_dtable"}},
                    {s.x, s.table, s.targets, s.lse, {grads->d_dloss, args->tokens, 4, 4, "d_dloss"}}));
    TRY(check_workspace(args->workspace, args->workspace_bytes, loss_grad_bytes(*args, *grads)));
    TRY(need_device());
    HIP_TRY(launch_loss_grad(*args, *grads, (hipStream_t)stream));
    return NSFPS_OK;
  });
}

}  // extern "C"
