#define DSDPA_T float
#include "dsdpa_cache_simt.inc"
