// Expert products of fp32 rows.
#include "expert_tile.h"

EL_FOR_TYPE(float, f32)
