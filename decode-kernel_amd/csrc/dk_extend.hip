// The extend (prefill) kernels of one head_dim (DK_HEAD_DIM, set by the build: 64, 128 or
// 256) and their symbol table.
#include "dk_extend.h"

#ifndef DK_HEAD_DIM
#error "compile once per head_dim with -DDK_HEAD_DIM=64, 128 or 256"
#endif

namespace dk {
namespace {
template <class T, int POOL>
const void* sym(bool cap) {
  return cap ? reinterpret_cast<const void*>(&dk_extend<T, DK_HEAD_DIM, POOL, true>)
             : reinterpret_cast<const void*>(&dk_extend<T, DK_HEAD_DIM, POOL, false>);
}
template <class T>
const void* sym_t(int pool, bool cap) {
  return pool == kPoolKv4   ? sym<T, kPoolKv4>(cap)
         : pool == kPoolFp8 ? sym<T, kPoolFp8>(cap)
                            : sym<T, kPoolSame>(cap);
}
}  // namespace

template <int D>
const void* extend_symbol(bool bf16, int pool, bool cap) {
  return bf16 ? sym_t<BF16>(pool, cap) : sym_t<F16>(pool, cap);
}
template const void* extend_symbol<DK_HEAD_DIM>(bool, int, bool);
}  // namespace dk
