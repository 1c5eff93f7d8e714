// Tensors that a Python binding holds as objects: lists of them, the operands of a layer norm (host code only).
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

using Read = int (*)(void*, void*);

// a tensor of fp32 or bf16 in CUDA memory, with its type's code
bool read_tensor(Read read, void* object, DlTensor* t, int32_t* dtype) {
  *t = DlTensor{};
  if (!object || read(object, t) != 0) return false;
  const bool f32 = t->code == DL_FLOAT && t->bits == 32, bf16 = t->code == DL_BFLOAT && t->bits == 16;
  *dtype = f32 ? MACE_F32 : MACE_BF16;
  return t->device_type == DL_CUDA && t->lanes == 1 && (f32 || bf16);
}
void* data_of(const DlTensor& t) { return static_cast<char*>(t.data) + t.byte_offset; }

// n rows of C contiguous channels, one stride apart
bool rows_of(const DlTensor& t, int64_t* n, int64_t* C, int64_t* stride) {
  if (t.ndim < 1) return false;
  *C = t.shape[t.ndim - 1];
  if (t.strides && t.strides[t.ndim - 1] != 1 && *C != 1) return false;
  *n = 1;
  *stride = *C;
  int64_t step = *C;  // from row to row where they are contiguous
  bool first = true;
  for (int32_t d = t.ndim - 2; d >= 0; --d) {
    const int64_t size = t.shape[d], s = t.strides ? t.strides[d] : step;
    if (size != 1 && first) *stride = s, first = false;
    else if (size != 1 && *n != 0 && s != *stride * *n) return false;
    *n *= size;
    step *= size;
  }
  return *C >= 1 && *C <= MACE_LAYER_NORM_MAX_CHANNELS && *n <= INT32_MAX && *stride >= 0;
}

}  // namespace

extern "C" int mace_tensor_list(int (*read)(void*, void*), int32_t count, void* const* objects, int32_t device,
                                void** data, int64_t* sizes, int32_t* dtypes) {
  if (!read || count < 0 || (count > 0 && (!objects || !data || !sizes || !dtypes)))
    return fail(MACE_ERR_BAD_ARG, "mace_tensor_list: bad arguments");
  for (int32_t i = 0; i < count; ++i) {
    DlTensor t;
    int32_t dtype;
    if (!read_tensor(read, objects[i], &t, &dtype) || t.device_id != device) return MACE_ERR_BAD_ARG;
    int64_t values = 1;
    bool dense = true;
    for (int32_t d = t.ndim - 1; d >= 0; --d) {
      if (t.shape[d] != 1 && t.strides && t.strides[d] != values) dense = false;
      values *= t.shape[d];
    }
    if (values != 0 && !dense) return MACE_ERR_BAD_ARG;
    data[i] = values ? data_of(t) : nullptr;
    sizes[i] = values;
    dtypes[i] = dtype;
  }
  return MACE_OK;
}

extern "C" int mace_list_items(void* (*get)(void*, intptr_t), void* list, int32_t count, void* none, void** objects) {
  int found = 0;
  for (int32_t i = 0; i < count; ++i) {
    objects[i] = get(list, i);
    if (!objects[i]) return -1;
    if (objects[i] == none) found = 1;
  }
  return found;
}

extern "C" int mace_norm_rows_read(int (*read)(void*, void*), void* x, void* dy, void* weight, void* bias,
                                   mace_norm_rows* rows) {
  if (!read || !x || !rows) return fail(MACE_ERR_BAD_ARG, "mace_norm_rows_read: bad arguments");
  mace_norm_rows r{};
  DlTensor t;
  int64_t C;
  if (!read_tensor(read, x, &t, &r.dtype) || !rows_of(t, &r.n, &C, &r.x_stride)) return MACE_ERR_BAD_ARG;
  r.C = (int32_t)C;
  r.device = t.device_id;
  r.x = data_of(t);
  if (!r.x && r.n > 0) return MACE_ERR_BAD_ARG;
  if (dy) {
    DlTensor g;
    int32_t dtype;
    int64_t n, c;
    if (!read_tensor(read, dy, &g, &dtype) || dtype != r.dtype || g.device_id != r.device || g.ndim != t.ndim ||
        !rows_of(g, &n, &c, &r.dy_stride))
      return MACE_ERR_BAD_ARG;
    for (int32_t d = 0; d < t.ndim; ++d)
      if (g.shape[d] != t.shape[d]) return MACE_ERR_BAD_ARG;
    r.dy = data_of(g);
    if (!r.dy && r.n > 0) return MACE_ERR_BAD_ARG;
  }
  r.param_dtype = r.dtype;
  void* const params[2] = {weight, bias};
  for (int k = 0; k < 2; ++k) {
    if (!params[k]) continue;
    DlTensor q;
    int32_t dtype;
    if (!read_tensor(read, params[k], &q, &dtype) || (dtype != r.dtype && dtype != MACE_F32) || q.device_id != r.device ||
        q.ndim != 1 || q.shape[0] != C || (q.strides && q.strides[0] != 1 && C != 1) || (k == 1 && weight && dtype != r.param_dtype))
      return MACE_ERR_BAD_ARG;
    r.param_dtype = dtype;
    void* const at = data_of(q);
    if (!at) return MACE_ERR_BAD_ARG;  // (a tensor without memory: null would stand for no parameter)
    (k == 0 ? r.weight : r.bias) = at;
  }
  *rows = r;
  return MACE_OK;
}

extern "C" int mace_norm_rows_forward(const mace_norm_rows* r, float eps, int32_t activation, void* y, void* stream) {
  if (!r) return fail(MACE_ERR_BAD_ARG, "mace_norm_rows_forward: bad arguments");
  return mace_layer_norm(r->dtype, r->x, r->x_stride, r->param_dtype, r->weight, r->bias, r->n, r->C, eps, activation, y, r->C,
                         stream);
}

extern "C" int mace_norm_rows_backward(const mace_norm_rows* r, float eps, int32_t activation, void* dx, void* dweight,
                                       void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!r) return fail(MACE_ERR_BAD_ARG, "mace_norm_rows_backward: bad arguments");
  return mace_layer_norm_grad(r->dtype, r->x, r->x_stride, r->dy, r->dy_stride, r->param_dtype, r->weight, r->bias, r->n, r->C,
                              eps, activation, dx, r->C, dweight, dbias, workspace, workspace_bytes, stream);
}
