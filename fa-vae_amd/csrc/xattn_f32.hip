// Cross attention, f32 elements: the kernels of xattn.h for this type.
#include "xattn_launch.h"

XATTN_INSTANTIATE(F32)
