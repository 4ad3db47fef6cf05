#define DSDPA_T __half
#include "dsdpa_few.inc"
