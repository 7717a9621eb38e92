// The gated feed-forward block's kernels in f32 (see gated_ffn_kernel.h).
#include "gated_ffn_kernel.h"

const srmi::FfnLaunch* srmi_ffn_f32() {
    static const srmi::FfnLaunch table = srmi::ffn_launches<SRMI_F32>();
    return &table;
}
