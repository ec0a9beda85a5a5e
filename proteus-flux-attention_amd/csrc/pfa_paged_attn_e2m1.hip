// One-token attention over e2m1 cells.
#include "pfa_paged_attn.h"

namespace pfa {
namespace paged {

void attend_e2m1(int qt, const AttendCall& a) {
  switch (qt) {
    case PFA_F32: return attend_by_width<PFA_F32, PFA_E2M1>(a);
    case PFA_BF16: return attend_by_width<PFA_BF16, PFA_E2M1>(a);
    default: return attend_by_width<PFA_F16, PFA_E2M1>(a);
  }
}

}  // namespace paged
}  // namespace pfa
