// The gated feed-forward block's kernels in f16 (see gated_ffn_kernel.h).
#include "gated_ffn_kernel.h"

const srmi::FfnLaunch* srmi_ffn_f16() {
    static const srmi::FfnLaunch table = srmi::ffn_launches<SRMI_F16>();
    return &table;
}
