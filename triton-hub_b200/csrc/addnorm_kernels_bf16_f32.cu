#define B200NORM_T __nv_bfloat16
#define B200NORM_R float
#define B200NORM_WIDE 2
#define B200NORM_GETTER addnorm_table_bf16_f32
#include "addnorm_kernels.inc"
