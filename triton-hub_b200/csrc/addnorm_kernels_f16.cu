#define B200NORM_T __half
#define B200NORM_R __half
#define B200NORM_WIDE 1
#define B200NORM_GETTER addnorm_table_f16
#include "addnorm_kernels.inc"
