// The gated feed-forward block's kernels in bf16 (see gated_ffn_kernel.h).
#include "gated_ffn_kernel.h"

const srmi::FfnLaunch* srmi_ffn_bf16() {
    static const srmi::FfnLaunch table = srmi::ffn_launches<SRMI_BF16>();
    return &table;
}
