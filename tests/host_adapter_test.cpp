// Host-only check of the C++ adapter: builds ops through the reference-shaped factories,
// checks object order, validation codes and the packer against a literal golden vector.
#include <cstdio>
#include <cstring>

#include <cstdlib>
#include <cstdio>
#include <string>

#include "../ml-drift_amd/host/mld_hip_ops.h"

using namespace mld_hip;

#define EXPECT(cond)                                              \
  do {                                                            \
    if (!(cond)) {                                                \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      return 1;                                                   \
    }                                                             \
  } while (0)

int main() {
  // common/task/weights_conversion_test.cc:50-91
  OHWI shape{4, 1, 1, 4};
  std::vector<uint8_t> src;
  for (int i = 0; i < 8; ++i) src.push_back((uint8_t)(((2 * i + 1) << 4) | (2 * i)));
  WeightsDescription d{};
  d.type = MLDHIP_UINT8;
  d.layout = MLDHIP_LAYOUT_OSPATIAL_IOGROUP_I4O4;
  d.output_group_size = 1;
  std::vector<uint8_t> packed;
  std::vector<int32_t> sums;
  EXPECT(RearrangeWeightsUInt4Packed(src.data(), shape, d, &packed, &sums).ok());
  const int order[16] = {0, 4, 8, 12, 1, 5, 9, 13, 2, 6, 10, 14, 3, 7, 11, 15};
  for (int i = 0; i < 8; ++i) EXPECT(packed[i] == (uint8_t)((order[2 * i] | (order[2 * i + 1] << 4)) ^ 0x88));
  EXPECT(sums[0] == 6 && sums[1] == 22 && sums[2] == -26 && sums[3] == -10);
  d.layout = MLDHIP_LAYOUT_OSPATIAL_IOGROUP_O4I4;
  Status st = RearrangeWeightsUInt4Packed(src.data(), shape, d, &packed, &sums);
  EXPECT(st.code == MLDHIP_UNIMPLEMENTED && st.message == "Unsupported layout");

  ExternalWeights w;
  w.shape = OHWI{14336, 1, 1, 4096};
  w.desc = GetFullyConnectedInt4WeightsDesc(w.shape);
  w.scale_zp_shape = OHWI{14336, 1, 1, 1};
  w.has_scale_tensor = true;
  HipOperation fc;
  EXPECT(CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, w,
                                             /*has_bias=*/true, 4, &fc)
             .ok());
  auto names = fc.GetSrcTensorsNames();
  EXPECT(names.size() == 4 && names[0] == "src_tensor" && names[1] == "weights" && names[2] == "weights_scale" &&
         names[3] == "biases");
  EXPECT(fc.UpdateParams(BHWC{1, 1, 5, 4096}).code == MLDHIP_OUT_OF_RANGE);
  EXPECT(fc.AddToQueue(nullptr).code == MLDHIP_FAILED_PRECONDITION);  // nothing bound: refused before any GPU call

  w.desc.output_group_size = 5;  // does not divide the slices
  HipOperation bad;
  st = CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, w,
                                           false, 1, &bad);
  EXPECT(st.code == MLDHIP_INVALID_ARGUMENT && !bad.valid());

  // runtime channel bounds: one more src object, "params", registered last; ringed uint4 weights are refused
  // as the reference refuses them (types under 8 bits, fully_connected.cc:1087-1092)
  w.desc = GetFullyConnectedInt4WeightsDesc(w.shape);
  ConvRuntimeCheckDesc rc_desc;
  rc_desc.src_end_ch_index = 1;
  rc_desc.dst_end_ch_index = 3;
  HipOperation bounded;
  EXPECT(CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, w,
                                             /*has_bias=*/true, 4, &bounded, rc_desc)
             .ok());
  names = bounded.GetSrcTensorsNames();
  EXPECT(names.size() == 5 && names[3] == "biases" && names[4] == "params");
  rc_desc.ring_o_offset_index = 0;
  rc_desc.ring_size = 14336;
  HipOperation ringed;
  st = CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, w,
                                           false, 1, &ringed, rc_desc);
  EXPECT(st.code == MLDHIP_INVALID_ARGUMENT && !ringed.valid());
  // ringed uint8 weights: a ring of 56 input rows under 20 src channels (fully_connected_test_util.cc:742-900)
  {
    ExternalWeights w8;
    w8.shape = OHWI{72, 1, 1, 56};
    w8.desc = GetFullyConnectedInt8WeightsDesc(w8.shape);
    w8.scale_zp_shape = OHWI{72, 1, 1, 1};
    w8.has_scale_tensor = true;
    ConvRuntimeCheckDesc ring;
    ring.ring_i_offset_index = 0;
    ring.src_end_ch_index = 1;
    ring.ring_size = 56;
    HipOperation ring_op;
    EXPECT(CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32, DataType::kFloat32, DataType::kFloat32, w8,
                                               /*has_bias=*/true, 1, &ring_op, ring, /*src_channels=*/20)
               .ok());
    names = ring_op.GetSrcTensorsNames();
    EXPECT(names.size() == 5 && names[4] == "params");
  }

  // FullyConnectedOI: the same op over output groups of one slice (fully_connected_oi_test_util.cc:109-111)
  ExternalWeights woi = w;
  woi.desc.output_group_size = 1;
  HipOperation oi;
  EXPECT(CreateFullyConnectedOI(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, woi,
                                /*has_bias=*/true, 4, &oi)
             .ok());
  names = oi.GetSrcTensorsNames();
  EXPECT(names.size() == 4 && names[1] == "weights" && names[3] == "biases");
  HipOperation not_oi;
  EXPECT(CreateFullyConnectedOI(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, w, true, 4, &not_oi)
             .code == MLDHIP_INVALID_ARGUMENT);

  // packed groups (gpu_model_builder_moe_util.cc:133-141, 214-224): batched weights, "params" last
  {
    ExternalWeights wp;
    wp.shape = OHWI{768, 128, 1, 2048};
    mldhip_fc_int4_weights_desc_reference(768, 2048, &wp.desc);
    wp.scale_zp_shape = OHWI{768, 128, 1, 64};
    wp.has_scale_tensor = true;
    ConvRuntimeCheckDesc rc_packed;
    rc_packed.packed_groups.params_offset = 0;
    rc_packed.packed_groups.num_groups = 128;
    rc_packed.packed_groups.max_group_size = 64;
    HipOperation grouped;
    EXPECT(CreateFullyConnectedExternalWeights(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, wp,
                                               /*has_bias=*/false, 512, &grouped, rc_packed)
               .ok());
    names = grouped.GetSrcTensorsNames();
    EXPECT(names.size() == 4 && names[1] == "weights" && names[2] == "weights_scale" && names[3] == "params");
  }

  // the mixture-of-experts FullyConnected: fully_connected.cc:1203-1213 registers batch_ids before the weights
  ExternalWeights we;
  we.shape = OHWI{768, 128, 1, 2048};
  we.desc = GetFullyConnectedInt4WeightsDesc(we.shape);
  we.scale_zp_shape = OHWI{768, 128, 1, 64};
  we.has_scale_tensor = true;
  HipOperation moe;
  EXPECT(CreateFullyConnectedWeightsBatchIds(CalculationsPrecision::kF32F16, DataType::kFloat16, DataType::kFloat16, we,
                                             /*has_bias=*/false, /*shared_src=*/true, 32, &moe)
             .ok());
  names = moe.GetSrcTensorsNames();
  EXPECT(names.size() == 4 && names[0] == "src_tensor" && names[1] == "batch_ids" && names[2] == "weights" &&
         names[3] == "weights_scale");
  EXPECT(moe.UpdateParams(BHWC{1, 8, 1, 2048}).ok());
  EXPECT(moe.UpdateParams(BHWC{2, 8, 1, 2048}).code == MLDHIP_UNIMPLEMENTED);

  HipOperation q;
  EXPECT(CreateQuantization(DataType::kFloat16, PackedType::kInt8C16, BHWC{1, 1, 2048, 2048}, false, true, &q).ok());
  EXPECT(q.GetDstTensorsNames().size() == 2 && q.GetDstTensorsNames()[1] == "dst_params");

  ExternalWeights w8;
  w8.shape = OHWI{8192, 1, 1, 2048};
  w8.desc = GetFullyConnectedInt8WeightsDesc(w8.shape);
  w8.scale_zp_shape = OHWI{8192, 1, 1, 1};
  EXPECT(SelectFullyConnectedRoute(w8, 1, true, false) == FcRoute::kFullyConnected);
  EXPECT(SelectFullyConnectedRoute(w8, 2048, true, false) == FcRoute::kQuantizedInt8);
  EXPECT(SelectFullyConnectedRoute(w8, 2048, true, true) == FcRoute::kFullyConnected);
  EXPECT(SelectFullyConnectedRoute(w, 512, false, false) == FcRoute::kFullyConnected);
  HipOperation conv;
  EXPECT(CreateConvInt8WithDequantization(DataType::kFloat16, w8.shape, GetConvolutionInt8WeightsDesc(w8.shape), false,
                                          false, 2048, &conv)
             .ok());
  EXPECT(conv.GetSrcTensorsNames().size() == 5 && conv.GetSrcTensorsNames()[2] == "params_tensor");

  // A layer from checkpoint files (samples/llm/llm_weights_loader.cc:29-71): int4 [4][8] with
  // nibbles 0..7 per row pattern, two scale groups of 4 input channels, written here by hand.
  {
    const char* tmp = std::getenv("TMPDIR");
    const std::string dir = std::string(tmp ? tmp : "/tmp") + "/";
    const std::string base = "mldhip_adapter_layer";
    std::vector<uint8_t> nib(4 * 8 / 2);
    for (int e = 0; e < 32; e += 2) nib[e / 2] = (uint8_t)(((e % 8) & 15) | ((((e + 1) % 8) - 8) & 15) << 4);
    std::vector<float> sc(4 * 2);
    for (int k = 0; k < 8; ++k) sc[k] = 0.5f + 0.25f * k;
    FILE* f = std::fopen((dir + base + ".weight").c_str(), "wb");
    EXPECT(f && std::fwrite(nib.data(), 1, nib.size(), f) == nib.size());
    std::fclose(f);
    f = std::fopen((dir + base + ".weight_quantized_scale").c_str(), "wb");
    EXPECT(f && std::fwrite(sc.data(), 4, sc.size(), f) == sc.size());
    std::fclose(f);
    LoadedFcWeights lw;
    EXPECT(LoadFcWeights(dir, base + ".weight", base, OHWI{4, 1, 1, 8}, 4, false, DataType::kFloat32, &lw).ok());
    EXPECT(lw.quantization_i_group_size == 4 && lw.weights.scale_zp_shape.i == 2 && !lw.weights.has_zero_point_tensor);
    EXPECT(lw.packed.size() == 16 && lw.scale.size() == 2 * 4 * 4 && lw.zero_point.empty());
    // row sums: elements e, e+1 of a row are (e % 8) and ((e+1) % 8) - 8: 0-7+2-5+4-3+6-1 = -4
    EXPECT(lw.weights_sum_i[0] == -4 && lw.weights_sum_i[3] == -4);
    // scale tensor [group][slice][4]: group 0 holds sc[o*2 + 0]
    const float* st32 = reinterpret_cast<const float*>(lw.scale.data());
    EXPECT(st32[0] == sc[0] && st32[1] == sc[2] && st32[4] == sc[1] && st32[7] == sc[7]);
    EXPECT(LoadFcWeights(dir, "no_such_file", base, OHWI{4, 1, 1, 8}, 4, false, DataType::kFloat32, &lw).code ==
           MLDHIP_NOT_FOUND);
    std::remove((dir + base + ".weight").c_str());
    std::remove((dir + base + ".weight_quantized_scale").c_str());
  }
  // a gated launch over unbound ops is refused before anything reaches the GPU
  EXPECT(AddToQueueGated(&fc, &fc, GateActivation::kSilu, nullptr, 0, nullptr).code == MLDHIP_INVALID_ARGUMENT);

  // between the projections: created, bound by name and shaped without a GPU
  {
    HipOperation op;
    QkNormRopeAttributes rope;
    rope.heads = 8;
    rope.kv_heads = 1;
    rope.head_dim = rope.rotary_dim = 256;
    EXPECT(CreateQkNormRope(DataType::kFloat16, rope, 4, &op).ok());
    EXPECT(op.GetSrcTensorsNames().size() == 3 && op.GetSrcTensorsNames()[2] == "positions" && op.GetDstTensorsNames()[1] == "dst_k");
    rope.norm = true;
    EXPECT(CreateQkNormRope(DataType::kFloat32, rope, 4, &op).ok() && op.GetSrcTensorsNames().size() == 5);
    rope.rotary_dim = 12;
    EXPECT(CreateQkNormRope(DataType::kFloat16, rope, 4, &op).code == MLDHIP_INVALID_ARGUMENT);
    Kv4Cache cache{/*kv_heads=*/1, /*head_dim=*/256, /*group_size=*/32, /*page_size=*/64, /*pages=*/10, /*sequences=*/2, /*pages_per_sequence=*/5};
    size_t bytes = 0;
    EXPECT(GetKv4CacheBytes(cache, &bytes).ok() && bytes == (size_t)10 * 64 * (256 + 4 * 8));
    EXPECT(CreateKv4Append(cache, DataType::kFloat16, 4, 2, &op).ok() && op.GetDstTensorsNames()[0] == "cache");
    EXPECT(CreateKv4Read(cache, DataType::kFloat32, 4, 2, &op).ok() && op.GetSrcTensorsNames()[0] == "cache");
    EXPECT(CreateKv4Attention(cache, 8, 0.0625f, true, 0, 4, 2, &op).ok() && op.GetSrcTensorsNames()[4] == "starts");
    EXPECT(op.UpdateParams(BHWC{1, 1, 4, 2048}).ok());
    EXPECT(op.UpdateParams(BHWC{1, 1, 5, 2048}).code == MLDHIP_OUT_OF_RANGE);
    EXPECT(CreateKv4Attention(cache, 8, 0.0f, true, 0, 4, 2, &op).code == MLDHIP_INVALID_ARGUMENT);
    cache.page_size = 48;
    EXPECT(GetKv4CacheBytes(cache, &bytes).code == MLDHIP_INVALID_ARGUMENT);
    EXPECT(CreateKv4Append(cache, DataType::kFloat16, 4, 2, &op).code == MLDHIP_INVALID_ARGUMENT);
  }
  std::printf("host adapter ok\n");
  return 0;
}
