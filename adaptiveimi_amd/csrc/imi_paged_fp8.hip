// Attention over pages of 8-bit floats (e4m3) with a power of two per block.
#include "imi_paged.hpp"

namespace imi {

int paged_attention_fp8(const imi_paged_attention_args* a, hipStream_t stream) { return run<Fp8>(a, stream); }

}  // namespace imi
