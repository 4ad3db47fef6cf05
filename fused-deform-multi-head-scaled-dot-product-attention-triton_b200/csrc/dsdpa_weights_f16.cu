#define DSDPA_T __half
#include "dsdpa_weights.inc"
