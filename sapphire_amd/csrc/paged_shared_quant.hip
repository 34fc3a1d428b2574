// paged_shared_quant.hip - the shared positions' kernels over quantized caches (paged_shared.h).
#include "paged_shared.h"

namespace sapphire {

bool launch_shared_quant(const void *args, const void *plan, hipStream_t s) {
    const AttnArgs &g = *static_cast<const AttnArgs *>(args);
    const SharedPlan &sp = *static_cast<const SharedPlan *>(plan);
    const int io = g.a.q.dtype;
#define SPH_FORM(CT, HD)                                                                      \
    if (g.a.c.dtype == CT && g.a.c.hd == HD) {                                                \
        if (io == DT_F32) launch_shared_form<CT, HD, false, false>(g, sp, s);                 \
        else if (io == DT_BF16) launch_shared_form<CT, HD, true, true>(g, sp, s);             \
        else launch_shared_form<CT, HD, true, false>(g, sp, s);                               \
    }
    SPH_FORM(DT_Q8_0, 64) SPH_FORM(DT_Q8_0, 128) SPH_FORM(DT_Q8_0, 256)
    SPH_FORM(DT_Q4_0, 64) SPH_FORM(DT_Q4_0, 128) SPH_FORM(DT_Q4_0, 256)
    return hip_ok(hipGetLastError(), "shared attention launch");
}

}  // namespace sapphire
