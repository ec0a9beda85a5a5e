// One-token attention over cells of the queries' own type.
#include "pfa_paged_attn.h"

namespace pfa {
namespace paged {

void attend_float(int qt, const AttendCall& a) {
  switch (qt) {
    case PFA_F32: return attend_by_width<PFA_F32, PFA_F32>(a);
    case PFA_BF16: return attend_by_width<PFA_BF16, PFA_BF16>(a);
    default: return attend_by_width<PFA_F16, PFA_F16>(a);
  }
}

}  // namespace paged
}  // namespace pfa
