#define B200NORM_T float
#define B200NORM_R float
#define B200NORM_WIDE 0
#define B200NORM_GETTER addnorm_table_f32
#include "addnorm_kernels.inc"
