#define B200NORM_T __nv_bfloat16
#define B200NORM_R __nv_bfloat16
#define B200NORM_WIDE 1
#define B200NORM_GETTER addnorm_table_bf16
#include "addnorm_kernels.inc"
