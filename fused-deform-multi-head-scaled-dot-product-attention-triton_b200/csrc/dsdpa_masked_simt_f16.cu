#define DSDPA_T __half
#include "dsdpa_masked_simt.inc"
