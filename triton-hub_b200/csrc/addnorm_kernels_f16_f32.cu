#define B200NORM_T __half
#define B200NORM_R float
#define B200NORM_WIDE 2
#define B200NORM_GETTER addnorm_table_f16_f32
#include "addnorm_kernels.inc"
