// K-g, the form for narrow rows (xent_narrow.h) of bfloat16
#include "xent_narrow.h"

XENT_NARROW(__bf16);
