// Addresses of many tensors of a Python framework at once, for operators that take lists (the AdamW step).  Asking 128 tensors for five
// properties each takes Python 30 us; the C table of the DLPack standard (`__dlpack_c_exchange_api__`, header version 1) has
// a function that describes one tensor object in some 20 ns.  The structures below are that standard's.
#include "common.h"

namespace {

struct DlTensor {
  void* data;
  int32_t device_type, device_id;            // 1: host, 2: CUDA
  int32_t ndim;
  uint8_t code, bits;                        // 2: float, 4: bfloat
  uint16_t lanes;
  int64_t* shape;
  int64_t* strides;                          // null: row-major
  uint64_t byte_offset;
};
using Describe = int (*)(void* object, DlTensor* out);

}  // namespace

extern "C" int b200tp_tensor_rows(void* describe, const int64_t* objects, int32_t count, int32_t dtype, int32_t device,
                                  b200tp_adamw_tensor* rows, int32_t column) {
  const Describe fn = reinterpret_cast<Describe>(describe);
  if (column < 0 || column > 2) return count;
  const uint8_t code = dtype == B200TP_BF16 ? 4 : 2, bits = dtype == B200TP_BF16 ? 16 : 32;
  for (int32_t i = 0; i < count; ++i) {
    DlTensor t;
    if (fn(reinterpret_cast<void*>(objects[i]), &t) != 0) return -2;
    if (t.code != code || t.bits != bits || t.lanes != 1) return i;
    if (device < 0 ? t.device_type != 1 : t.device_type != 2 || t.device_id != device) return i;
    int64_t numel = 1;
    bool row_major = true;
    for (int32_t k = t.ndim - 1; k >= 0; --k) {
      if (t.strides != nullptr && t.shape[k] != 1 && t.strides[k] != numel) row_major = false;
      numel *= t.shape[k];
    }
    if (numel != rows[i].numel || (!row_major && numel != 0)) return i;
    char* data = static_cast<char*>(t.data) + t.byte_offset;
    if (column == 0) rows[i].param = data;
    else if (column == 1) rows[i].grad = data;
    else rows[i].param_out = data;
  }
  return -1;
}
