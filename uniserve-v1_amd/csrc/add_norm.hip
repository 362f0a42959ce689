// SPDX-License-Identifier: Apache-2.0
//
// add_norm on gfx950 (include/uniserve_add_norm.h states the operator): a row is read once into
// registers, joined, and normed there; means and squares are summed in FP32 over a lane's elements, the
// wavefront's lanes and, where a row has several wavefronts, their sums through LDS in a fixed order.
#include "add_norm.hpp"
#include "extents.hpp"

namespace uniserve {
namespace add_norm {
namespace {

int64_t size_of(int32_t dtype) { return dtype == UNISERVE_DTYPE_F32 ? 4 : 2; }

int32_t run(const uniserve_add_norm_call *call, void *stream) {
  const int64_t rows = call->rows, width = call->width;
  if (rows < 0 || width <= 0) return UNISERVE_REFUSE(call, "add_norm needs non-negative rows and a positive width");
  if (width > UNISERVE_ADD_NORM_MAX_WIDTH)
    return UNISERVE_REFUSE(call, "add_norm serves rows of up to %d elements", UNISERVE_ADD_NORM_MAX_WIDTH);
  if (call->dtype != UNISERVE_DTYPE_BF16 && call->dtype != UNISERVE_DTYPE_F16 && call->dtype != UNISERVE_DTYPE_F32)
    return UNISERVE_REFUSE(call, "add_norm norms bf16, f16 or f32 rows");
  const bool streams = call->residual != nullptr || call->total != nullptr;
  if (streams && call->total_dtype != call->dtype && call->total_dtype != UNISERVE_DTYPE_F32)
    return UNISERVE_REFUSE(call, "add_norm's residual and total are of the input's type or f32");
  const bool vectors = call->post != nullptr || call->channels != nullptr || call->weight != nullptr;
  if (vectors && call->vector_dtype != call->dtype && call->vector_dtype != UNISERVE_DTYPE_F32)
    return UNISERVE_REFUSE(call, "add_norm's vectors are of the input's type or f32");
  if (call->norm != UNISERVE_NORM_RMS && call->norm != UNISERVE_NORM_LAYER)
    return UNISERVE_REFUSE(call, "add_norm's norm is rms or layer");
  if (call->norm == UNISERVE_NORM_RMS && (call->bias != nullptr || call->post_bias != nullptr))
    return UNISERVE_REFUSE(call, "add_norm's rms norm has no bias");
  if (call->post_bias != nullptr && call->post == nullptr) return UNISERVE_REFUSE(call, "add_norm's post_bias comes with post");
  if (!(call->eps >= 0.0f)) return UNISERVE_REFUSE(call, "add_norm's eps is not negative");
  if (rows == 0) return 0;  // (arrays of no rows may have no address)
  if ((call->weight == nullptr) != (call->out == nullptr) || (call->bias != nullptr && call->weight == nullptr))
    return UNISERVE_REFUSE(call, "add_norm's weight and out come together, its bias with them");
  if (call->input == nullptr || (call->out == nullptr && call->total == nullptr))
    return UNISERVE_REFUSE(call, "add_norm needs an input and an output");
  // A single row has no stride to go by, an absent array neither.
  const auto stride_of = [&](const void *array, int64_t stride) { return array != nullptr && rows > 1 ? stride : width; };
  AddNormParams p{};
  p.x_stride = stride_of(call->input, call->input_row_stride);
  p.residual_stride = stride_of(call->residual, call->residual_row_stride);
  p.total_stride = stride_of(call->total, call->total_row_stride);
  p.out_stride = stride_of(call->out, call->out_row_stride);
  p.gate_stride = call->gate != nullptr && rows > 1 ? call->gate_stride : 0;
  for (const int64_t stride : {p.x_stride, p.residual_stride, p.total_stride, p.out_stride}) {
    if (stride < width) return UNISERVE_REFUSE(call, "add_norm's row strides are shorter than its rows");
    if (stride > kMostElements / rows) return UNISERVE_REFUSE(call, "add_norm's arrays are too large");
  }
  if (p.gate_stride < 0) return UNISERVE_REFUSE(call, "add_norm's gate stride is negative");
  if (p.gate_stride > kMostElements / rows) return UNISERVE_REFUSE(call, "add_norm's arrays are too large");
  const int64_t element = size_of(call->dtype), wide = size_of(call->total_dtype), vector = size_of(call->vector_dtype);
  const Extent input = extent(call->input, rows, width, p.x_stride, element);
  const Extent residual = extent(call->residual, rows, width, p.residual_stride, wide);
  const Extent total = extent(call->total, rows, width, p.total_stride, wide);
  const Extent out = extent(call->out, rows, width, p.out_stride, element);
  // A lane reads its elements of a row before it writes any of them: an output over the very elements of an
  // input is in place.
  const auto in_place = [](const Extent &a, const Extent &b) {
    return a.first == b.first && a.bytes == b.bytes && (a.stride == b.stride || a.rows == 1);
  };
  for (const Extent &to : {total, out}) {
    for (const Extent &from : {input, residual})
      if (overlap(to, from) && !in_place(to, from))
        return UNISERVE_REFUSE(call, "add_norm's output overlaps one of its inputs in part");
    for (const void *array : {call->post, call->post_bias, call->channels, call->weight, call->bias})
      if (overlap(to, extent(array, 1, width, width, vector)))
        return UNISERVE_REFUSE(call, "add_norm's output overlaps one of its vectors");
    if (overlap(to, extent(call->gate, rows, 1, p.gate_stride, element)))
      return UNISERVE_REFUSE(call, "add_norm's output overlaps its gate");
  }
  if (overlap(total, out)) return UNISERVE_REFUSE(call, "add_norm's outputs overlap");

  p.x = call->input, p.residual = call->residual, p.total = call->total, p.out = call->out;
  p.post = call->post, p.post_bias = call->post_bias, p.channels = call->channels;
  p.weight = call->weight, p.bias = call->bias;
  p.gate = call->gate;
  p.rows = rows, p.width = static_cast<int32_t>(width);
  p.vector_f32 = call->vector_dtype == UNISERVE_DTYPE_F32;
  p.layer = call->norm == UNISERVE_NORM_LAYER;
  p.eps = call->eps, p.offset = call->offset, p.scale = call->scale, p.residual_scale = call->residual_scale;
  p.inverse_width = 1.0f / static_cast<float>(width);
  const bool total_f32 = streams && call->total_dtype == UNISERVE_DTYPE_F32;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (call->dtype == UNISERVE_DTYPE_F32) launch<F32, F32>(p, s);
  else if (call->dtype == UNISERVE_DTYPE_F16) total_f32 ? launch<F16, F32>(p, s) : launch<F16, F16>(p, s);
  else total_f32 ? launch<Bf16, F32>(p, s) : launch<Bf16, Bf16>(p, s);
  return launched(call, "add_norm");
}

}  // namespace
}  // namespace add_norm
}  // namespace uniserve

extern "C" int32_t uniserve_add_norm(const uniserve_add_norm_call *call, void *stream) {
  return uniserve::guarded(call, [&]() { return uniserve::add_norm::run(call, stream); });
}
