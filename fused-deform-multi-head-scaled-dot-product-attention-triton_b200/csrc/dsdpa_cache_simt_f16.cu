#define DSDPA_T __half
#include "dsdpa_cache_simt.inc"
