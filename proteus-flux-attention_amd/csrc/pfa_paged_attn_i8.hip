// One-token attention over int8 cells.
#include "pfa_paged_attn.h"

namespace pfa {
namespace paged {

void attend_i8(int qt, const AttendCall& a) {
  switch (qt) {
    case PFA_F32: return attend_by_width<PFA_F32, PFA_I8>(a);
    case PFA_BF16: return attend_by_width<PFA_BF16, PFA_I8>(a);
    default: return attend_by_width<PFA_F16, PFA_I8>(a);
  }
}

}  // namespace paged
}  // namespace pfa
