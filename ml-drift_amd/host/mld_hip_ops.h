// C++ host-side mirror of the reference's operator interface for the quantized
// fully-connected path, on top of the C-ABI (include/mldhip.h).
//
// Names, argument meaning and error behaviour follow the reference so that a builder /
// backend written against ML Drift's types maps one to one:
//   WeightsDescription, OHWI, BHWC            common/task/weights_layout.h, common/shape.h
//   ExternalWeights                            common/task/gpu_operation.h:354-363
//   CreateFullyConnectedExternalWeights        common/kernels/fully_connected.h:155-161
//   CreateFullyConnectedWeightsBatchIds        common/kernels/fully_connected.cc:1174-1216
//   CreateFullyConnectedOI                     common/kernels/fully_connected_oi.h:80-86
//   CreateQuantization                         common/kernels/quantize_and_dequantize.h:68-73
//   ClOperation::{SetSrcTensor, SetDstTensor, UpdateParams, AddToQueue}   cl/cl_operation.h:44-129
//   GpuModelBuilder::FullyConnectedInt4/8ExternalWeights (dispatcher)     common/gpu_model_builder.cc:1548-1725
// Status is a small stand-in for absl::Status carrying the same code numbers.
#ifndef MLD_HIP_OPS_H_
#define MLD_HIP_OPS_H_

#include <cstdint>
#include <memory>
#include <string>
#include <utility>
#include <vector>

#include "../../include/mldhip.h"

namespace mld_hip {

struct Status {
  int code = MLDHIP_OK;
  std::string message;
  bool ok() const { return code == MLDHIP_OK; }
  static Status FromCode(int c) { return c == MLDHIP_OK ? Status{} : Status{c, mldhip_last_error()}; }
};

struct OHWI {
  int o = 0, h = 1, w = 1, i = 0;
};
struct BHWC {
  int b = 1, h = 1, w = 1, c = 0;
};
enum class CalculationsPrecision { kF32 = 0, kF32F16 = 1, kF16 = 2 };
enum class DataType { kFloat16 = 1, kFloat32 = 2, kUint8 = 5, kInt8 = 6, kInt32 = 10, kUint4 = 15 };
enum class PackedType {  // common/data_type.h:48-58
  kUint8C4 = 1, kInt8C4 = 2, kUint8W4C4 = 3, kInt8W4C4 = 4, kInt8C16 = 5, kUint8C16 = 6, kInt4C32 = 7, kUint4C32 = 8
};

using WeightsDescription = mldhip_weights_desc;

inline WeightsDescription GetFullyConnectedInt8WeightsDesc(const OHWI& shape) {
  WeightsDescription d;
  mldhip_fc_int8_weights_desc(shape.o, shape.i, &d);
  return d;
}
inline WeightsDescription GetFullyConnectedInt4WeightsDesc(const OHWI& shape) {
  WeightsDescription d;
  // (batched weights, h = the weights batch, take the same description: the packers put the matrices
  // of an output group one after the other)
  mldhip_fc_int4_weights_desc(shape.o, shape.i, &d);
  return d;
}
inline WeightsDescription GetConvolutionInt8WeightsDesc(const OHWI& shape) {
  WeightsDescription d;
  mldhip_conv_int8_weights_desc(shape.o, shape.i, &d);
  return d;
}
inline size_t GetTotalElementsCountForLayout(const WeightsDescription& d, const OHWI& s) {
  size_t n = 0;
  mldhip_total_elements(&d, s.o, s.h, s.w, s.i, &n);
  return n;
}

// Host packers, same names as common/task/weights_conversion.h.
inline Status RearrangeWeightsInt8AsUint8(const int8_t* w, const OHWI& s, const WeightsDescription& d,
                                          std::vector<uint8_t>* dst, int shift = 128, unsigned pad = 128u) {
  dst->resize(GetTotalElementsCountForLayout(d, s));
  return Status::FromCode(
      mldhip_rearrange_int8_as_uint8(w, s.o, s.h, s.w, s.i, &d, dst->data(), dst->size(), shift, pad));
}
inline Status RearrangeWeightsInt8AsUint4(const int8_t* w, const OHWI& s, const WeightsDescription& d,
                                          std::vector<uint8_t>* dst, int shift = 8, unsigned pad = 8u) {
  dst->resize(GetTotalElementsCountForLayout(d, s) / 2);
  return Status::FromCode(
      mldhip_rearrange_int8_as_uint4(w, s.o, s.h, s.w, s.i, &d, dst->data(), dst->size(), shift, pad));
}
inline Status RearrangeWeightsUInt4Packed(const uint8_t* w, const OHWI& s, const WeightsDescription& d,
                                          std::vector<uint8_t>* dst, std::vector<int32_t>* weights_sum_i,
                                          unsigned pad = 8u, bool swap_dims = false) {
  dst->resize(GetTotalElementsCountForLayout(d, s) / 2);
  if (weights_sum_i->size() < (size_t)s.o) weights_sum_i->resize(s.o);
  return Status::FromCode(mldhip_rearrange_uint4_packed(w, s.o, s.h, s.w, s.i, &d, dst->data(), dst->size(),
                                                        weights_sum_i->data(), weights_sum_i->size(), pad, swap_dims));
}

// Shape/type of the quantized weights of one layer; device buffers are the caller's
// (ExternalWeights holds non-owning descriptors in the reference as well).
struct ExternalWeights {
  WeightsDescription desc{};
  OHWI shape;
  OHWI scale_zp_shape{1, 1, 1, 1};  // (o,1,1,groups); (1,1,1,1) = scalar
  bool has_scale_tensor = false;
  bool has_zero_point_tensor = false;
  float scalar_scale = 1.0f;
  bool has_scalar_zero_point = false;
  float scalar_zero_point = 0.0f;
};

// ConvRuntimeCheckDesc (common/task/gpu_operation.h:384-412): indices into the int32 "params"
// object of the op, -1 = not set.
struct ConvRuntimeCheckDesc {
  int src_end_ch_index = -1;
  int dst_end_ch_index = -1;
  int ring_o_offset_index = -1;
  int ring_i_offset_index = -1;
  int ring_size = 0;
  bool HasValues() const {
    return src_end_ch_index >= 0 || dst_end_ch_index >= 0 || ring_o_offset_index >= 0 || ring_i_offset_index >= 0;
  }
  // for batched weights: the tokens of the source row are sorted by weight matrix, sizes and offsets
  // of the groups are read from the params object (gpu_operation.h:396-406); num_groups == 0 = not set
  struct PackedGroups {
    int params_offset = 0;  // [num_groups] sizes, then [num_groups] offsets
    int num_groups = 0;     // the batch size of the weights (ExternalWeights::shape.h)
    int max_group_size = 0;
  };
  PackedGroups packed_groups;
};

// A node executor: what ClOperation is to a GPUOperation in the reference.
class HipOperation {
 public:
  HipOperation() = default;
  explicit HipOperation(mldhip_op* op) : op_(op, &mldhip_op_destroy) {}
  HipOperation(HipOperation&&) = default;  // move-only, like GPUOperation
  HipOperation& operator=(HipOperation&&) = default;

  std::vector<std::string> GetSrcTensorsNames() const {
    std::vector<std::string> r;
    for (int i = 0; i < mldhip_op_src_count(op_.get()); ++i) r.emplace_back(mldhip_op_src_name(op_.get(), i));
    return r;
  }
  std::vector<std::string> GetDstTensorsNames() const {
    std::vector<std::string> r;
    for (int i = 0; i < mldhip_op_dst_count(op_.get()); ++i) r.emplace_back(mldhip_op_dst_name(op_.get(), i));
    return r;
  }
  Status SetSrcTensor(int index, const void* device_ptr, size_t bytes) {
    return Status::FromCode(mldhip_op_set_src(op_.get(), index, device_ptr, bytes));
  }
  Status SetDstTensor(int index, void* device_ptr, size_t bytes) {
    return Status::FromCode(mldhip_op_set_dst(op_.get(), index, device_ptr, bytes));
  }
  // UpdateParams: re-evaluates everything that depends on the runtime tensor shape.
  Status UpdateParams(const BHWC& src_shape) {
    return Status::FromCode(mldhip_op_set_shape(op_.get(), src_shape.b, src_shape.h, src_shape.w));
  }
  Status AddToQueue(void* hip_stream) { return Status::FromCode(mldhip_op_launch(op_.get(), hip_stream)); }
  const char* kernel_name() const { return mldhip_op_kernel_name(op_.get()); }
  bool valid() const { return op_ != nullptr; }
  mldhip_op* handle() const { return op_.get(); }

 private:
  std::unique_ptr<mldhip_op, void (*)(mldhip_op*)> op_{nullptr, &mldhip_op_destroy};
};

namespace detail {
inline mldhip_fc_desc FcDescOf(CalculationsPrecision precision, DataType src_type, DataType dst_type,
                               const ExternalWeights& weights, bool has_bias, int max_tokens,
                               const ConvRuntimeCheckDesc& runtime_check = {}, int src_channels = 0, int dst_channels = 0);
}  // namespace detail

// CreateFullyConnectedWeightsBatchIds (common/kernels/fully_connected.h, .cc:1174-1216): the
// FullyConnected of a mixture-of-experts layer.  weights.shape.h = number of weight matrices;
// src objects: src_tensor, batch_ids, weights, [weights_scale, weights_zero_point,] [biases].
// UpdateParams(BHWC(1, ids, tokens per id, c)) sets the dst shape; `shared_src`: the source tensor
// has one row that every id reads (its H is 1), else one row per id.
inline Status CreateFullyConnectedWeightsBatchIds(CalculationsPrecision precision, DataType src_type,
                                                  DataType dst_type, const ExternalWeights& weights, bool has_bias,
                                                  bool shared_src, int max_tokens, HipOperation* result,
                                                  const ConvRuntimeCheckDesc& runtime_check = {}) {
  const mldhip_fc_desc d = detail::FcDescOf(precision, src_type, dst_type, weights, has_bias, max_tokens, runtime_check);
  mldhip_op* op = nullptr;
  const int rc = mldhip_fc_batch_ids_create(&d, weights.shape.h, shared_src ? 1 : 0, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

// With runtime channel bounds or a ring offset the op takes a last src object "params" (int32 values on
// the device).  Ringed weights (fully_connected.cc:411-471, 676-706): the tensor along the ringed axis
// has channels of its own, which the reference reads from the `src` / `dst` descriptors it is handed:
// `src_channels` with ring_i_offset_index (weights.shape.i = the ring), `dst_channels` with
// ring_o_offset_index (weights.shape.o = the ring); 0 = the weights' own.
inline Status CreateFullyConnectedExternalWeights(CalculationsPrecision precision, DataType src_type,
                                                  DataType dst_type, const ExternalWeights& weights, bool has_bias,
                                                  int max_tokens, HipOperation* result,
                                                  const ConvRuntimeCheckDesc& runtime_check = {}, int src_channels = 0,
                                                  int dst_channels = 0) {
  const mldhip_fc_desc d = detail::FcDescOf(precision, src_type, dst_type, weights, has_bias, max_tokens, runtime_check,
                                            src_channels, dst_channels);
  mldhip_op* op = nullptr;
  const int rc = mldhip_fc_create(&d, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

// CreateFullyConnectedOI (common/kernels/fully_connected_oi.cc:530-583): the FullyConnected over
// weights with the output slice outermost, linear_i4o4 = dst_s * src_slices + src_s (:122-133),
// which is kOSpatialIOGroupI4O4 with output_group_size = 1 (what the reference's tests pass,
// tests/fully_connected_oi_test_util.cc:109-111, 256-258).  Same objects and arithmetic as
// CreateFullyConnectedExternalWeights; a description with another group size is refused here.
inline Status CreateFullyConnectedOI(CalculationsPrecision precision, DataType src_type, DataType dst_type,
                                     const ExternalWeights& weights, bool has_bias, int max_tokens,
                                     HipOperation* result, const ConvRuntimeCheckDesc& runtime_check = {}) {
  if (weights.desc.output_group_size != 1) return Status::FromCode(MLDHIP_INVALID_ARGUMENT);
  return CreateFullyConnectedExternalWeights(precision, src_type, dst_type, weights, has_bias, max_tokens, result,
                                             runtime_check);
}

inline mldhip_fc_desc detail::FcDescOf(CalculationsPrecision precision, DataType src_type, DataType dst_type,
                                       const ExternalWeights& weights, bool has_bias, int max_tokens,
                                       const ConvRuntimeCheckDesc& runtime_check, int src_channels, int dst_channels) {
  mldhip_fc_desc d{};
  d.src_channels = src_channels;
  d.dst_channels = dst_channels;
  d.has_runtime_check = 1;
  d.src_end_ch_index = runtime_check.src_end_ch_index;
  d.dst_end_ch_index = runtime_check.dst_end_ch_index;
  d.ring_o_offset_index = runtime_check.ring_o_offset_index;
  d.ring_i_offset_index = runtime_check.ring_i_offset_index;
  d.ring_size = runtime_check.ring_size;
  d.packed_params_offset = runtime_check.packed_groups.params_offset;
  d.packed_num_groups = runtime_check.packed_groups.num_groups;
  d.packed_max_group_size = runtime_check.packed_groups.max_group_size;
  d.precision = (int)precision;
  d.src_type = (int)src_type;
  d.dst_type = (int)dst_type;
  d.o = weights.shape.o;
  d.i = weights.shape.i;
  d.weights = weights.desc;
  d.scale_o = weights.has_scale_tensor ? weights.scale_zp_shape.o : 1;
  d.scale_i = weights.has_scale_tensor ? weights.scale_zp_shape.i : 1;
  d.scalar_scale = weights.scalar_scale;
  d.has_zero_point_tensor = weights.has_zero_point_tensor;
  d.has_scalar_zero_point = weights.has_scalar_zero_point;
  d.scalar_zero_point = weights.scalar_zero_point;
  d.has_bias = has_bias;
  d.max_tokens = max_tokens;
  return d;
}

inline Status CreateQuantization(DataType src_type, PackedType dst_type, const BHWC& shape, bool calculate_sum,
                                 bool symmetric, HipOperation* result) {
  mldhip_quant_desc d{(int)src_type, (int)dst_type, shape.c, calculate_sum, symmetric, shape.b * shape.h * shape.w, 0};
  mldhip_op* op = nullptr;
  const int rc = mldhip_quantization_create(&d, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

inline Status CreateConvInt8WithDequantization(DataType dst_type, const OHWI& weights_shape,
                                               const WeightsDescription& weights_desc, bool has_zero_point,
                                               bool has_bias, int max_tokens, HipOperation* result) {
  mldhip_conv_int8_desc d{};
  d.src_packed_type = mldhip_conv_int8_src_type();
  d.dst_type = (int)dst_type;
  d.o = weights_shape.o;
  d.i = weights_shape.i;
  d.weights = weights_desc;
  d.has_zero_point = has_zero_point;
  d.has_bias = has_bias;
  d.max_tokens = max_tokens;
  mldhip_op* op = nullptr;
  const int rc = mldhip_conv_int8_create(&d, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

// Between the q / k / v projections and the o projection (no counterparts in the reference's FullyConnected path; include/mldhip.h:
// arithmetic, layouts, objects).  Norms of the query and key heads and the rotation by position; `frequencies` as for
// mldhip_qk_norm_rope_desc (read here, need not outlive the call).
struct QkNormRopeAttributes {
  int heads = 0, kv_heads = 0, head_dim = 0, rotary_dim = 0;
  double base = 10000.0;
  const double* frequencies = nullptr;
  bool interleaved = false;
  bool norm = false;
  float eps = 1e-6f, weight_offset = 0.0f;
};
inline Status CreateQkNormRope(DataType tensor_type, const QkNormRopeAttributes& attr, int max_tokens, HipOperation* result) {
  const mldhip_qk_norm_rope_desc d{(int)tensor_type, attr.heads, attr.kv_heads, attr.head_dim, attr.rotary_dim, attr.base, attr.frequencies,
                                   attr.interleaved, attr.norm, attr.eps, attr.weight_offset, max_tokens};
  mldhip_op* op = nullptr;
  const int rc = mldhip_qk_norm_rope_create(&d, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

// The key / value cache of 4-bit codes in pages, and the ops over it.
using Kv4Cache = mldhip_kv4_cache_desc;
inline Status GetKv4CacheBytes(const Kv4Cache& cache, size_t* bytes) { return Status::FromCode(mldhip_kv4_cache_bytes(&cache, bytes)); }
inline Status CreateKv4Append(const Kv4Cache& cache, DataType src_type, int max_tokens, int max_new_tokens, HipOperation* result) {
  mldhip_op* op = nullptr;
  const int rc = mldhip_kv4_append_create(&cache, (int)src_type, max_tokens, max_new_tokens, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}
inline Status CreateKv4Read(const Kv4Cache& cache, DataType dst_type, int max_tokens, int max_new_tokens, HipOperation* result) {
  mldhip_op* op = nullptr;
  const int rc = mldhip_kv4_read_create(&cache, (int)dst_type, max_tokens, max_new_tokens, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}
inline Status CreateKv4Attention(const Kv4Cache& cache, int heads, float scale, bool causal, int window, int max_tokens,
                                 int max_new_tokens, HipOperation* result) {
  const mldhip_kv4_attention_desc d{cache, heads, scale, causal, window, max_tokens, max_new_tokens};
  mldhip_op* op = nullptr;
  const int rc = mldhip_kv4_attention_create(&d, &op);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  *result = HipOperation(op);
  return {};
}

// One launch for FullyConnected nodes that read the same tensor (q/k/v, gate/up); the caller
// falls back to AddToQueue per node when the status is FAILED_PRECONDITION.
inline Status AddToQueueFused(const std::vector<HipOperation*>& ops, void* hip_stream) {
  std::vector<mldhip_op*> handles;
  for (HipOperation* op : ops) handles.push_back(op->handle());
  return Status::FromCode(mldhip_fc_launch_fused(handles.data(), (int)handles.size(), hip_stream));
}

// gelu_tanh(gate(x)) * up(x) / silu(gate(x)) * up(x) in the launch of the two projections: the
// Linear, Linear, GeluTanhMul / SiluMul nodes of the sample's FFLayer
// (samples/llm/gemma3_model_builder.cc:1141-1147) as one.  kFailedPrecondition: keep the three nodes.
enum class GateActivation { kGeluTanh = MLDHIP_GATE_GELU_TANH, kSilu = MLDHIP_GATE_SILU };
inline Status AddToQueueGated(HipOperation* gate, HipOperation* up, GateActivation activation, void* dst_device_ptr,
                              size_t dst_bytes, void* hip_stream) {
  return Status::FromCode(
      mldhip_fc_launch_gated(gate->handle(), up->handle(), (int)activation, dst_device_ptr, dst_bytes, hip_stream));
}

// One linear layer read from the LLM sample's checkpoint files, as host buffers ready to upload:
// what LlmWeightsLoader::GetWeightsInt4 / GetWeightsInt8 (samples/llm/llm_weights_loader.cc:29-117)
// assemble through LlmFileTensorLoader.  `weights` carries the description and shapes that
// CreateFullyConnectedExternalWeights takes; the tensors are in the activation type.
struct LoadedFcWeights {
  ExternalWeights weights;
  int quantization_i_group_size = 0;
  std::vector<uint8_t> packed;          // "weights"
  std::vector<uint8_t> scale;           // "weights_scale", tensor bytes
  std::vector<uint8_t> zero_point;      // "weights_zero_point", empty without a zero-point file
  std::vector<int32_t> weights_sum_i;   // for the int8 x int8 route
};

inline Status LoadFcWeights(const std::string& weights_directory, const std::string& w_name,
                            const std::string& base_name, const OHWI& weights_shape, int weight_bits, bool swap_dims,
                            DataType tensor_type, LoadedFcWeights* out) {
  mldhip_checkpoint_fc info;
  int rc = mldhip_checkpoint_fc_probe(weights_directory.c_str(), w_name.c_str(), base_name.c_str(), weights_shape.o,
                                      weights_shape.i, weight_bits, &info);
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  const size_t elem = tensor_type == DataType::kFloat16 ? 2 : 4;
  out->packed.assign(info.weights_bytes, 0);
  out->scale.assign(info.scale_elements * elem, 0);
  out->zero_point.assign(info.has_zero_point ? info.scale_elements * elem : 0, 0);
  out->weights_sum_i.assign(weights_shape.o, 0);
  rc = mldhip_checkpoint_fc_read(weights_directory.c_str(), w_name.c_str(), base_name.c_str(), &info, swap_dims ? 1 : 0,
                                 (int)tensor_type, out->packed.data(), out->packed.size(), out->scale.data(),
                                 info.has_zero_point ? out->zero_point.data() : nullptr, out->scale.size(),
                                 out->weights_sum_i.data());
  if (rc != MLDHIP_OK) return Status::FromCode(rc);
  out->quantization_i_group_size = info.group_size;
  out->weights.desc = info.weights;
  out->weights.shape = weights_shape;
  out->weights.scale_zp_shape = OHWI{weights_shape.o, 1, 1, info.scale_i};
  out->weights.has_scale_tensor = true;
  out->weights.has_zero_point_tensor = info.has_zero_point != 0;
  return Status{};
}

// One graph node: operation + the ids of its inputs/outputs in the caller's tensor table,
// in the reference's order (common/gpu_model.h:38-60).
struct GpuNode {
  HipOperation gpu_operation;
  std::vector<int> inputs;
  std::vector<int> outputs;
  std::string name;
};

// The route the builder takes for a quantized FullyConnected
// (GpuModelBuilder::FullyConnectedInt4/8ExternalWeights, common/gpu_model_builder.cc:1548-1725),
// restated for this device:
//   kFullyConnected   one FC node over the packed FC weights (any token count: streaming GEMV
//                     for a few tokens, fused dequantize+MFMA GEMM beyond; the reference would
//                     emit WeightsConverter + float ConvGeneric there)
//   kQuantizedInt8    Quantize -> int8 conv (+ Dequantization), available for per-channel int8
//                     weights with weights_sum_i when 8-bit convolutions are not disallowed
enum class FcRoute { kFullyConnected, kQuantizedInt8 };

inline FcRoute SelectFullyConnectedRoute(const ExternalWeights& w, int tokens, bool has_weights_sum_i,
                                         bool disallow_8bit_convs) {
  const bool grouped = w.scale_zp_shape.i != 1;
  const bool int8_weights = w.desc.type == MLDHIP_UINT8 || w.desc.type == MLDHIP_INT8;
  if (mldhip_fc_is_recommended((int)CalculationsPrecision::kF32F16, tokens)) return FcRoute::kFullyConnected;
  if (!grouped && int8_weights && has_weights_sum_i && !disallow_8bit_convs) return FcRoute::kQuantizedInt8;
  return FcRoute::kFullyConnected;
}

}  // namespace mld_hip

#endif  // MLD_HIP_OPS_H_
