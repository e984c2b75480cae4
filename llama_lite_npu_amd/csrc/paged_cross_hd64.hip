// The head dim 64 build of paged_cross.hip.
#define LITEKV_CROSS 1
#define LITEKV_HD 64
#include "paged_prefill.hip"
