// Expert products of bf16 rows.
#include "expert_tile.h"

EL_FOR_TYPE(__hip_bfloat16, bf16)
