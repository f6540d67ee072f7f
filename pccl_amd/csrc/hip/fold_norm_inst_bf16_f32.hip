// fold_norm_inst_bf16_f32.hip -- instantiates the norms around a block for bf16 rows, f32 parameters.
#include "fold_norm_kernel.h"

namespace pccl_dev {
PCCL_DEFINE_FOLD_NORM(PCCL_BF16, true)
}  // namespace pccl_dev
