// A layer's key/value cache in 8 bits as the kernels take it (kv8.h), shared with the op bindings.
#pragma once

#include <stdint.h>

namespace mx {

// Keys and values apart: codes e4m3 [pages, Hkv, block, D], exponent bytes [pages, Hkv, block / 16]; table int32
// [slots, maxp]: position p of slot s lies in page table[s][p / block] at row p % block.
struct Kv8Pages {
  uint8_t *k, *v, *ke, *ve;
  const int32_t* table;
  int slots, maxp, block, pages, Hkv;
};

}  // namespace mx
