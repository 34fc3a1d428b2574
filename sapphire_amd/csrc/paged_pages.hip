// paged_pages.hip - attention of one new token per sequence over the pages that a list per K/V head names. The kernels are
// the attention's over all pages (paged_attention.h); a walk goes along the list and looks each page up by it.
#include "paged_attention.h"

namespace sapphire {

int launch_paged_pages_attention(const PagedAttn &a, hipStream_t s) { return launch_attention<LIST>(a, s); }

}  // namespace sapphire
