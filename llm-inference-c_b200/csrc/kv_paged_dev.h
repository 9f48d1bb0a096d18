// kv_paged_dev.h - what other device code of this library takes from a paged
// cache's handle (kv_paged.cu) beyond include/kv_paged.h.
#ifndef KV_PAGED_DEV_H
#define KV_PAGED_DEV_H

#include "kv_paged.h"

// Device address of the handle's error bits (kv_paged_error reads and clears
// them), for a step that brings them back with its results.
const int *kv_paged_error_word(const KvPaged *kv);

#endif
