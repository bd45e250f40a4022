// f32 kernels of rel_attn (rel_attn_body.h): head widths up to 32, 64 and 128
#include "rel_attn_body.h"

int rel_run_f32(const RelP& p, int what, int nw, hipStream_t st) {
    return p.D <= 32 ? pick_nw<float, 32>(p, what, nw, st) : p.D <= 64 ? pick_nw<float, 64>(p, what, nw, st) : pick_nw<float, 128>(p, what, nw, st);
}
