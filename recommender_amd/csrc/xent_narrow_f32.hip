// K-g, the form for narrow rows (xent_narrow.h) of 32-bit floats
#include "xent_narrow.h"

XENT_NARROW(float);
