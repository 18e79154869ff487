// Decode attention kernels over the 4-bit cache for one head_dim (DK_HEAD_DIM, set by the build:
// 64, 128 or 256) and their symbol table.
#include "dk_kv4.h"

#ifndef DK_HEAD_DIM
#error "compile once per head_dim with -DDK_HEAD_DIM=64, 128 or 256"
#endif

namespace dk {
namespace {
template <class T, int HP, bool CAP, int NW>
const void* sym(bool balanced) {
  return balanced ? reinterpret_cast<const void*>(&dk_kv4_balanced<T, DK_HEAD_DIM, HP, CAP, NW>)
                  : reinterpret_cast<const void*>(&dk_kv4_split<T, DK_HEAD_DIM, HP, CAP, NW>);
}
template <class T, int HP>
const void* sym_hp(bool cap, int waves, bool balanced) {
  if (waves != 4) return nullptr;
  return cap ? sym<T, HP, true, 4>(balanced) : sym<T, HP, false, 4>(balanced);
}
template <class T>
const void* sym_t(int hp, bool cap, int waves, bool balanced) {
  switch (hp) {
    case 4: return sym_hp<T, 4>(cap, waves, balanced);
    case 8: return sym_hp<T, 8>(cap, waves, balanced);
    case 16: return sym_hp<T, 16>(cap, waves, balanced);
    default: return nullptr;
  }
}
}  // namespace

template <int D>
const void* kv4_symbol(bool bf16, int hp, bool cap, int waves, bool balanced) {
  return bf16 ? sym_t<BF16>(hp, cap, waves, balanced) : sym_t<F16>(hp, cap, waves, balanced);
}
template const void* kv4_symbol<DK_HEAD_DIM>(bool, int, bool, int, bool);
}  // namespace dk
