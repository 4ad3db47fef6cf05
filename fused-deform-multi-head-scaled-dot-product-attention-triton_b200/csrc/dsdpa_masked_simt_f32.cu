#define DSDPA_T float
#include "dsdpa_masked_simt.inc"
