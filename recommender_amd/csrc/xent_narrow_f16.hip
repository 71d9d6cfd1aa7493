// K-g, the form for narrow rows (xent_narrow.h) of half precision
#include "xent_narrow.h"

XENT_NARROW(_Float16);
