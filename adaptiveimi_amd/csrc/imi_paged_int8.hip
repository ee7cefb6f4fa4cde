// Attention over pages of 8-bit whole numbers with a power of two per block.
#include "imi_paged.hpp"

namespace imi {

int paged_attention_int8(const imi_paged_attention_args* a, hipStream_t stream) { return run<Int8>(a, stream); }

}  // namespace imi
