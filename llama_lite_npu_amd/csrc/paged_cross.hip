// Attention of packed rows over another sequence's keys in pages (an encoder's states): paged_prefill.hip with every row
// seeing all of them, and the C ABI of that.
#define LITEKV_CROSS 1
#include "paged_prefill.hip"
