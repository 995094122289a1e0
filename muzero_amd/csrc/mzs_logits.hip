/*
 * mzs_logits.hip — initial inference that writes the policy head's logits (mzs_initial_logits).  Part of libmzsearch.so.
 */
#include <hip/hip_runtime.h>

#include "mzs_inference.h"

namespace mzs {

infer_kernel_t pick_logits_kernel(bool vision) {
    if (vision) return k_inference<kInferInitial, true, true>;
    return k_inference<kInferInitial, false, true>;
}

}  // namespace mzs
