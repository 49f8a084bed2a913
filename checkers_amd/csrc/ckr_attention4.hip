// checkers_amd/csrc/ckr_attention4.hip — attention over a cache in 4 bits: the kernels of
// ckr_attention.h for CKR_F4.
#include "ckr_attention.h"

namespace ckr {

hipError_t attend_four(const AttnArg& a, const Cut& c, int dtype, hipStream_t s) {
    return dtype == CKR_BF16 ? launch_attend_dim<ElemBF16, ElemF4>(a, c, s) : launch_attend_dim<ElemF16, ElemF4>(a, c, s);
}

}  // namespace ckr
