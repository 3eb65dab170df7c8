// sym_b200 -- C-ABI of the microscaled operators (include/sym_b200.h): checks
// of the arguments, the caller's device kept as it was, and the launches of
// the thin CUDA layer. Every call is asynchronous on the caller's stream,
// allocates nothing on the device and lets no exception out.
#include "sb_cuda.h"
#include "sym_b200.h"

#include <cstdint>
#include <cstdio>
#include <initializer_list>

namespace {

static_assert(sizeof(sb_mx) == sizeof(sbc_mx), "the two descriptors are one layout");

int fail(sb_error *err, const char *code, const char *message) {
  if (err) {
    std::snprintf(err->code, sizeof err->code, "%s", code);
    std::snprintf(err->message, sizeof err->message, "%s", message);
    err->offset = -1;
  }
  return 1;
}

int status(sb_error *err, const char *what, int rc) {
  if (rc == 0)
    return 0;
  char text[256];
  if (rc == SBC_EINVAL || rc == SBC_EUNSUPPORTED) {
    std::snprintf(text, sizeof text, "%s: the sizes or pointers do not fit the kernel", what);
    return fail(err, "invalid_view", text);
  }
  std::snprintf(text, sizeof text, "%s: %s", what, sbc_error_string(rc));
  return fail(err, "backend_failure", text);
}

/// Makes `device` current for the call and the caller's device afterwards.
class OnDevice {
public:
  explicit OnDevice(int device) {
    rc_ = sbc_get_device(&before_);
    if (!rc_ && before_ != device) {
      rc_ = sbc_set_device(device);
      moved_ = !rc_;
    }
  }
  ~OnDevice() {
    if (moved_)
      sbc_set_device(before_);
  }
  int rc() const { return rc_; }

private:
  int before_ = 0, rc_ = 0;
  bool moved_ = false;
};

bool aligned(uint64_t p) { return p != 0 && p % 16 == 0; }

/// NULL, or what is wrong with a matrix.
const char *wrong(const sb_mx *q) {
  if (!q)
    return "a microscaled matrix is missing";
  if (q->format != SBC_MXFP4 && q->format != SBC_MXINT8)
    return "the format is mxfp4 (0) or mxint8 (1)";
  if (q->rows <= 0 || q->cols <= 0)
    return "a microscaled matrix has at least one row and one column";
  // offsets of codes and values stay far inside 64 bits
  if (q->rows > (int64_t{1} << 40) || q->cols > (int64_t{1} << 40) || q->rows > (int64_t{1} << 56) / q->cols)
    return "a microscaled matrix is too large";
  if (!aligned(q->codes) || !aligned(q->scales))
    return "codes and scales start on 16-byte boundaries";
  if (q->device < 0)
    return "codes and scales live on a CUDA device";
  return nullptr;
}

const sbc_mx *C(const sb_mx *q) { return reinterpret_cast<const sbc_mx *>(q); }

bool known(int32_t dtype) { return dtype >= SBC_F32 && dtype <= SBC_BF16; }

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t code_bytes(int64_t rows, int64_t cols) { return rows * ((cols + 31) / 32) * 16; }
int64_t scale_bytes(int64_t rows, int64_t cols) { return (rows + 127) / 128 * ((cols + 127) / 128) * 512; }

/// A wait that ran out in an earlier call's kernel is reported by the device's
/// next product, as for the transfers with asynchronous completion, or on request
/// (sb_mx_status).
int earlier_fault(int32_t device, sb_error *err) {
  if (sbc_mx_take_fault(device))
    return fail(err, "backend_failure",
                "a bounded wait ran out in an earlier microscaled product; that product's output is incomplete");
  return 0;
}

} // namespace

extern "C" {

int sb_mx_quantize(const void *x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, const sb_mx *along,
                   const sb_mx *across, void *stream, sb_error *err) {
  if (!along && !across)
    return fail(err, "invalid_options", "nothing to write");
  for (const sb_mx *q : {along, across}) {
    if (!q)
      continue;
    if (const char *w = wrong(q))
      return fail(err, "invalid_view", w);
  }
  if (!x || rows <= 0 || cols <= 0 || row_stride < 0)
    return fail(err, "invalid_view", "x needs at least one row and one column, and rows no less than 0 apart");
  if (!known(dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  if ((along && (along->rows != rows || along->cols != cols)) ||
      (across && (across->rows != cols || across->cols != rows)))
    return fail(err, "invalid_view", "the extents differ from those of x");
  if (across && (across->format != SBC_MXFP4 || (along && along->format != SBC_MXFP4)))
    return fail(err, "typed_unsupported", "blocks along the rows are mxfp4");
  if (along && across && along->device != across->device)
    return fail(err, "device_mismatch", "the two results live on different devices");
  OnDevice on((along ? along : across)->device);
  if (on.rc())
    return status(err, "set device", on.rc());
  return status(err, "quantize",
                sbc_mx_quantize(x, dtype, rows, cols, row_stride, C(along), C(across), stream));
}

int sb_mx_dequantize(const sb_mx *q, void *out, int32_t dtype, int32_t transpose, void *stream, sb_error *err) {
  if (const char *w = wrong(q))
    return fail(err, "invalid_view", w);
  if (!out)
    return fail(err, "invalid_view", "out is missing");
  if (!known(dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  if (transpose && q->format != SBC_MXFP4)
    return fail(err, "typed_unsupported", "transposed values are those of mxfp4");
  OnDevice on(q->device);
  if (on.rc())
    return status(err, "set device", on.rc());
  return status(err, "dequantize", sbc_mx_dequantize(C(q), out, dtype, transpose, stream));
}

int sb_mx_matmul(const sb_mx *a, const sb_mx *b, void *y, int32_t dtype, void *stream, sb_error *err) {
  for (const sb_mx *q : {a, b})
    if (const char *w = wrong(q))
      return fail(err, "invalid_view", w);
  if (a->format != SBC_MXFP4 || b->format != SBC_MXFP4)
    return fail(err, "typed_unsupported", "products are those of mxfp4 matrices");
  if (a->cols != b->cols)
    return fail(err, "invalid_view", "a [m, k] and b [n, k] need the same k");
  if (a->device != b->device)
    return fail(err, "device_mismatch", "a and b live on different devices");
  if (!y)
    return fail(err, "invalid_view", "y is missing");
  if (!known(dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  OnDevice on(a->device);
  if (on.rc())
    return status(err, "set device", on.rc());
  if (earlier_fault(a->device, err))
    return 1;
  return status(err, "matmul", sbc_mx_product(C(a), nullptr, 0, 0, C(b), y, dtype, 0, stream));
}

int sb_mx_status(int32_t device, sb_error *err) {
  if (device < 0)
    return fail(err, "invalid_view", "devices are numbered from 0");
  return earlier_fault(device, err);
}

int sb_mx_linear_workspace(int64_t rows, int64_t n, int64_t k, int32_t device, int64_t *bytes, sb_error *err) {
  if (rows <= 0 || n <= 0 || k <= 0 || !bytes || rows > (int64_t{1} << 56) / k)
    return fail(err, "invalid_view", "extents are at least 1");
  OnDevice on(device);
  if (on.rc())
    return status(err, "set device", on.rc());
  *bytes = sbc_mx_fuses_quantize(rows, n, k) ? 0 : up256(code_bytes(rows, k)) + scale_bytes(rows, k);
  return 0;
}

int sb_mx_linear(const void *x, int32_t x_dtype, int64_t rows, int64_t row_stride, const sb_mx *weight, void *y,
                 int32_t y_dtype, void *workspace, int64_t workspace_bytes, void *stream, sb_error *err) {
  if (const char *w = wrong(weight))
    return fail(err, "invalid_view", w);
  if (weight->format != SBC_MXFP4)
    return fail(err, "typed_unsupported", "products are those of mxfp4 matrices");
  if (!x || !y || rows <= 0 || row_stride < 0 || rows > (int64_t{1} << 56) / weight->cols)
    return fail(err, "invalid_view", "x needs at least one row, and rows no less than 0 apart; y is needed");
  if (!known(x_dtype) || !known(y_dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  OnDevice on(weight->device);
  if (on.rc())
    return status(err, "set device", on.rc());
  if (earlier_fault(weight->device, err))
    return 1;
  const int64_t k = weight->cols;
  sbc_mx q{nullptr, nullptr, rows, k, SBC_MXFP4, weight->device};
  if (sbc_mx_fuses_quantize(rows, weight->rows, k))
    return status(err, "linear", sbc_mx_product(&q, x, x_dtype, row_stride, C(weight), y, y_dtype, 0, stream));
  const int64_t codes = up256(code_bytes(rows, k)), scales = scale_bytes(rows, k);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < codes + scales)
    return fail(err, "insufficient_capacity", "the workspace is smaller than sb_mx_linear_workspace asks for, or not aligned");
  q.codes = workspace;
  q.scales = static_cast<uint8_t *>(workspace) + codes;
  if (const int rc = sbc_mx_quantize(x, x_dtype, rows, k, row_stride, &q, nullptr, stream))
    return status(err, "quantize", rc);
  return status(err, "linear", sbc_mx_product(&q, nullptr, 0, 0, C(weight), y, y_dtype, 1, stream));
}

int sb_silu_mul(const void *gate, int64_t gate_stride, const void *up, int64_t up_stride, int32_t dtype, int64_t rows,
                int64_t cols, int32_t device, void *h, const sb_mx *gate_q, const sb_mx *up_q, void *stream,
                sb_error *err) {
  if (!gate || !up || !h || rows <= 0 || cols <= 0 || gate_stride < 0 || up_stride < 0)
    return fail(err, "invalid_view", "gate, up and h have at least one row and one column");
  if (!known(dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  if (!gate_q != !up_q)
    return fail(err, "invalid_options", "both inputs are kept or neither");
  if (gate_q) {
    for (const sb_mx *q : {gate_q, up_q}) {
      if (const char *w = wrong(q))
        return fail(err, "invalid_view", w);
      if (q->format != SBC_MXINT8 || q->rows != rows || q->cols != cols)
        return fail(err, "invalid_view", "the kept inputs are mxint8 of the extents of gate");
      if (q->device != device)
        return fail(err, "device_mismatch", "the kept inputs live on another device");
    }
  }
  OnDevice on(device);
  if (on.rc())
    return status(err, "set device", on.rc());
  return status(err, "silu_mul",
                sbc_silu_mul(gate, gate_stride, up, up_stride, dtype, rows, cols, h, C(gate_q), C(up_q), stream));
}

int sb_silu_mul_backward(const void *dh, int64_t dh_stride, int32_t dtype, const sb_mx *gate_q, const sb_mx *up_q,
                         void *dgate, int64_t dgate_stride, void *dup, int64_t dup_stride, void *stream,
                         sb_error *err) {
  for (const sb_mx *q : {gate_q, up_q})
    if (const char *w = wrong(q))
      return fail(err, "invalid_view", w);
  if (gate_q->format != SBC_MXINT8 || up_q->format != SBC_MXINT8 || gate_q->rows != up_q->rows ||
      gate_q->cols != up_q->cols)
    return fail(err, "invalid_view", "the kept inputs are mxint8 of the same extents");
  if (gate_q->device != up_q->device)
    return fail(err, "device_mismatch", "the kept inputs live on different devices");
  // rows of dgate and dup may not overlap each other
  if (!dh || !dgate || !dup || dh_stride < 0 ||
      (gate_q->rows > 1 && (dgate_stride < gate_q->cols || dup_stride < gate_q->cols)))
    return fail(err, "invalid_view", "dh, dgate and dup have the extents of gate");
  if (!known(dtype))
    return fail(err, "typed_unsupported", "values are float32, float16 or bfloat16");
  OnDevice on(gate_q->device);
  if (on.rc())
    return status(err, "set device", on.rc());
  return status(err, "silu_mul_backward",
                sbc_silu_mul_backward(dh, dh_stride, dtype, C(gate_q), C(up_q), dgate, dgate_stride, dup, dup_stride,
                                      stream));
}

} // extern "C"
