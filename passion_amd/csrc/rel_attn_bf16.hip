// bf16 kernels of rel_attn (rel_attn_body.h): head widths up to 32, 64 and 128
#include "rel_attn_body.h"

int rel_run_bf16(const RelP& p, int what, int nw, hipStream_t st) {
    return p.D <= 32 ? pick_nw<bf16_t, 32>(p, what, nw, st) : p.D <= 64 ? pick_nw<bf16_t, 64>(p, what, nw, st) : pick_nw<bf16_t, 128>(p, what, nw, st);
}
