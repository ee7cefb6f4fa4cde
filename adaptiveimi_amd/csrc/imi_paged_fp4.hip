// Attention over pages of 4-bit floats (e2m1) with a power of two per block.
#include "imi_paged.hpp"

namespace imi {

int paged_attention_fp4(const imi_paged_attention_args* a, hipStream_t stream) { return run<Fp4>(a, stream); }

}  // namespace imi
