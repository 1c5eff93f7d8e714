// Lists of tensors that a Python binding holds as objects (host code only).
#include "common.cuh"

using namespace mace;

namespace {

// A tensor as DLPack's C interface lays it out (dlpack.h, version 1).
struct DlTensor {
  void* data;
  int32_t device_type, device_id;
  int32_t ndim;
  uint8_t code, bits;  // of a value's type
  uint16_t lanes;
  const int64_t* shape;
  const int64_t* strides;  // in values; null: contiguous
  uint64_t byte_offset;
};
static_assert(sizeof(DlTensor) == 48, "the layout of DLPack's tensor on 64-bit hosts");

constexpr int32_t DL_CUDA = 2;
constexpr uint8_t DL_FLOAT = 2, DL_BFLOAT = 4;

}  // namespace

extern "C" int mace_tensor_list(int (*read)(void*, void*), int32_t count, void* const* objects, int32_t device,
                                void** data, int64_t* sizes, int32_t* dtypes) {
  if (!read || count < 0 || (count > 0 && (!objects || !data || !sizes || !dtypes)))
    return fail(MACE_ERR_BAD_ARG, "mace_tensor_list: bad arguments");
  for (int32_t i = 0; i < count; ++i) {
    DlTensor t{};
    if (!objects[i] || read(objects[i], &t) != 0) return MACE_ERR_BAD_ARG;
    const bool f32 = t.code == DL_FLOAT && t.bits == 32, bf16 = t.code == DL_BFLOAT && t.bits == 16;
    if (t.device_type != DL_CUDA || t.device_id != device || t.lanes != 1 || !(f32 || bf16)) return MACE_ERR_BAD_ARG;
    int64_t values = 1;
    bool dense = true;
    for (int32_t d = t.ndim - 1; d >= 0; --d) {
      if (t.shape[d] != 1 && t.strides && t.strides[d] != values) dense = false;
      values *= t.shape[d];
    }
    if (values != 0 && !dense) return MACE_ERR_BAD_ARG;
    data[i] = values ? static_cast<char*>(t.data) + t.byte_offset : nullptr;
    sizes[i] = values;
    dtypes[i] = f32 ? MACE_F32 : MACE_BF16;
  }
  return MACE_OK;
}
