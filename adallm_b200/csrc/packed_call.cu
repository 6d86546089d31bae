// ada_call: entries of many arguments with the arguments as one array of 64-bit words, for bindings
// whose cost a call goes by its arguments (ctypes converts thirty in 4-7 us, one packed buffer in 1.5).
#include <string.h>

#include "common.cuh"

namespace {
template <typename T>
T* at(int64_t w) { return reinterpret_cast<T*>(static_cast<uintptr_t>(w)); }
float real(int64_t w) {
  double d;
  memcpy(&d, &w, 8);
  return static_cast<float>(d);
}
int i32(int64_t w) { return static_cast<int>(w); }
// 32-bit arguments out of range would be other numbers: refused
bool fits(const int64_t* a, const char* kinds) {
  for (int i = 0; kinds[i]; ++i)
    if (kinds[i] == 'i' && a[i] != static_cast<int32_t>(a[i])) return false;
  return true;
}
}  // namespace

extern "C" int ada_call(int entry, const int64_t* a) {
  if (!a) return ADA_ERR_INVALID_ARG;
  switch (entry) {
    case ADA_CALL_STEP_METADATA:
      if (!fits(a, "ppipqipqpiqpppppppp")) return ADA_ERR_UNSUPPORTED;
      return ada_step_metadata(at<int32_t>(a[0]), at<int32_t>(a[1]), i32(a[2]), at<int32_t>(a[3]), a[4], i32(a[5]),
                               at<int32_t>(a[6]), a[7], at<int32_t>(a[8]), i32(a[9]), a[10], at<int64_t>(a[11]),
                               at<int32_t>(a[12]), at<int32_t>(a[13]), at<int32_t>(a[14]), at<int32_t>(a[15]),
                               at<int32_t>(a[16]), at<unsigned>(a[17]), at<void>(a[18]));
    case ADA_CALL_ROTARY:
      if (!fits(a, "ppqqpqqppqiiipqiiip")) return ADA_ERR_UNSUPPORTED;
      return ada_rotary(at<int64_t>(a[0]), at<void>(a[1]), a[2], a[3], at<void>(a[4]), a[5], a[6], at<void>(a[7]),
                        at<void>(a[8]), a[9], i32(a[10]), i32(a[11]), i32(a[12]), at<float>(a[13]), a[14], i32(a[15]),
                        i32(a[16]), i32(a[17]), at<void>(a[18]));
    case ADA_CALL_KV4_STORE:
      if (!fits(a, "ppqqpqqpqqpqiiipqiipppqqqiddip")) return ADA_ERR_UNSUPPORTED;
      return ada_kv4_store(at<int64_t>(a[0]), at<void>(a[1]), a[2], a[3], at<void>(a[4]), a[5], a[6], at<void>(a[7]),
                           a[8], a[9], at<void>(a[10]), a[11], i32(a[12]), i32(a[13]), i32(a[14]), at<float>(a[15]),
                           a[16], i32(a[17]), i32(a[18]), at<int32_t>(a[19]), at<uint8_t>(a[20]), at<uint8_t>(a[21]),
                           a[22], a[23], a[24], i32(a[25]), real(a[26]), real(a[27]), i32(a[28]), at<void>(a[29]));
    case ADA_CALL_KV4_READ:
      if (!fits(a, "ppqqqiiipqddppip")) return ADA_ERR_UNSUPPORTED;
      return ada_kv4_read(at<uint8_t>(a[0]), at<uint8_t>(a[1]), a[2], a[3], a[4], i32(a[5]), i32(a[6]), i32(a[7]),
                          at<int32_t>(a[8]), a[9], real(a[10]), real(a[11]), at<void>(a[12]), at<void>(a[13]),
                          i32(a[14]), at<void>(a[15]));
    case ADA_CALL_KV4_PAGED_DECODE:
      if (!fits(a, "piqqppqqqpqipiiiiidddipiqqpqp")) return ADA_ERR_UNSUPPORTED;
      return ada_kv4_paged_decode(at<void>(a[0]), i32(a[1]), a[2], a[3], at<uint8_t>(a[4]), at<uint8_t>(a[5]), a[6],
                                  a[7], a[8], at<int32_t>(a[9]), a[10], i32(a[11]), at<int32_t>(a[12]), i32(a[13]),
                                  i32(a[14]), i32(a[15]), i32(a[16]), i32(a[17]), real(a[18]), real(a[19]),
                                  real(a[20]), i32(a[21]), at<void>(a[22]), i32(a[23]), a[24], a[25], at<void>(a[26]),
                                  static_cast<size_t>(a[27]), at<void>(a[28]));
    case ADA_CALL_KV4_PAGED_PREFILL:
      if (!fits(a, "piqqppqqqpqippiqiiiiidddipiqqpqpp")) return ADA_ERR_UNSUPPORTED;
      return ada_kv4_paged_prefill(at<void>(a[0]), i32(a[1]), a[2], a[3], at<uint8_t>(a[4]), at<uint8_t>(a[5]), a[6],
                                   a[7], a[8], at<int32_t>(a[9]), a[10], i32(a[11]), at<int32_t>(a[12]),
                                   at<int32_t>(a[13]), i32(a[14]), a[15], i32(a[16]), i32(a[17]), i32(a[18]),
                                   i32(a[19]), i32(a[20]), real(a[21]), real(a[22]), real(a[23]), i32(a[24]),
                                   at<void>(a[25]), i32(a[26]), a[27], a[28], at<void>(a[29]), static_cast<size_t>(a[30]),
                                   at<unsigned>(a[31]), at<void>(a[32]));
    default:
      return ADA_ERR_INVALID_ARG;
  }
}
