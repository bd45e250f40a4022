// What the host side and the kernels of rel_attn share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "common.h"

struct RelP {
    const void *q, *k, *v, *dout, *o;     // q [B][Nq][H][D], k, v [B][Nk][Hkv][D] by strides; dout, o contiguous
    long qs[3], ks[3], vs[3];             // strides of (batch, token, head) in elements
    void *out, *dq, *dk, *dv;             // contiguous
    float *lse, *delta;                   // [B][H][Nq]; log2 domain, +inf: a row without a key
    const uint8_t* mask;                  // [B][Nk], 0: masked; NULL: none
    const float* e;                       // [H][nd] bias by offset, log2 units
    const void* table;                    // [nb][H], where few queries read it directly
    const int* buckets;                   // [nd]; NULL: an offset is its own bucket
    float* slab;                          // the table's partial gradients (LINE: rows of slab_len, else the dense sums); NULL: not wanted
    long slab_len;
    int QC, KC, parts;                    // dense sums: queries and keys of one pass (whole copies of the cells), parts of the passes
    float *po, *pm, *pl;                  // split forward: [nsplit][B][H][Nq](D), f32
    int B, Nq, Nk, H, Hkv, D;
    int gd, gh, gw, vol, nd, omax, q0, nb, tdt;
    int bias, pack, few, nsplit, ksplit;  // few: few query rows (forward), the bias read straight from the table; nsplit: parts of the keys (forward, dQ); ksplit: of the queries (dK, dV)
    float c, scale;                       // c = scale * log2(e)
};

// one table entry in log2 units: an entry at or below -1e30 (a type's lowest value, -inf) excludes the pair, a bucket outside the table has no bias
__device__ __forceinline__ float rel_log2_bias(const void* table, int tdt, int bucket, int nb, int head, int H) {
    if (bucket < 0 || bucket >= nb) return 0.f;
    const long at = (long)bucket * H + head;
    const float t = tdt == PASSION_BF16 ? (float)static_cast<const bf16_t*>(table)[at] : static_cast<const float*>(table)[at];
    return t <= -1e30f ? -INFINITY : fminf(t * 1.4426950408889634f, 3.0e38f) + (t != t ? t : 0.f);
}

// what: 0 forward, 1 dQ, 2 dK, dV (LINE: and the table's partials), 3 the dense sums of the table's gradient; nw: wavefronts a workgroup (1, 2 or 4)
int rel_run_bf16(const RelP& p, int what, int nw, hipStream_t st);
int rel_run_f32(const RelP& p, int what, int nw, hipStream_t st);
