// The extend (prefill) kernels over a 4-bit cache of one head_dim (DK_HEAD_DIM, set by the build: 64,
// 128 or 256) and their symbol table.
#include "dk_extend_kv4.h"

#ifndef DK_HEAD_DIM
#error "compile once per head_dim with -DDK_HEAD_DIM=64, 128 or 256"
#endif

namespace dk {
namespace {
template <class T>
const void* sym(bool cap) {
  return cap ? reinterpret_cast<const void*>(&dk_extend_kv4<T, DK_HEAD_DIM, true>)
             : reinterpret_cast<const void*>(&dk_extend_kv4<T, DK_HEAD_DIM, false>);
}
}  // namespace

template <int D>
const void* extend_kv4_symbol(bool bf16, bool cap) {
  return bf16 ? sym<BF16>(cap) : sym<F16>(cap);
}
template const void* extend_kv4_symbol<DK_HEAD_DIM>(bool, bool);
}  // namespace dk
