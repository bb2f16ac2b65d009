// Expert products of fp16 rows.
#include "expert_tile.h"

EL_FOR_TYPE(__half, f16)
