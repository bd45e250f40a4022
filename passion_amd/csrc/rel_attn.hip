// Attention with a learned relative position bias, forward and backward: host side and the small kernels (the large ones: rel_attn_body.h).
//
// Tokens lie in raster order on a grid (gd, gh, gw); token t sits at cell t mod (gd gh gw) (further modalities repeat the grid), query i is token
// q_start + i.  With o(i, j) the index of cell_i - cell_j among the (2 gd - 1)(2 gh - 1)(2 gw - 1) offsets:
//     s_ij = scale q_i . k_j + table[buckets[o(i, j)]][head]       (masked keys and entries at or below -1e30 are excluded)
//     p_i = softmax_j(s_ij), out_i = sum_j p_ij v_j                 (a row with nothing left: 0)
// backward, from the saved row log-sum-exp, the probabilities formed again (only the table's gradient keeps partial sums: over a grid one f32 a pair of cells and head, as
// large as a head's scores where every cell holds one token, and up to the batch times that while it is small; over a 1D raster 1/32 of the scores of all heads):
//     delta_i = dout_i . out_i,  dS = p (dout v^T - delta),  dq = scale dS k,  dk = scale dS^T q,  dv = p^T dout,  dtable[c] = sum over pairs of bucket c of dS
// The reference's SelfAttention (code/models/mmformer.py:192-227) has learned absolute positions instead; its tokens are such a grid.
//
// Two backward kernels as in flash_attn.hip: query-major (dq) and key-major (dk, dv: the heads that share a key / value head sum in registers), and the table's sums
// (rel_attn_body.h); all free of atomics.
//
// Bound: long sequences by the matrix pipe and the vector arithmetic per score (exponential, bias, conversions), one token by the latency of a chain of loads.  Measured, bf16
// (kernel times; they follow the clock, 331 to 372 us for the first from box to box):
//   8000 x 8000 tokens, 8 heads of 128 on 4, 1D table: forward 329 us (797 TF), dq 509 (772 TF), dk / dv / diagonal sums 797 (658 TF), fold 42;
//   4 x 2048 x 2048, 8 heads of 64, 8^3 cells, 30 % of the keys masked: forward 74, dq 84, dk / dv 93, the table's dense sums 80, fold 17 us;
//   4 x 1 x 6000, 8 heads of 64 on 2: 9.5 + 6 us (12.4 MB of cache).
#include "common.h"
#include "passion_hip.h"
#include "rel_attn.h"

namespace {

constexpr int MAX_WG = 1 << 21;         // workgroups along x of the small kernels' launches: below 2^32 threads, past which a launch is cut off without an error
constexpr int BOX_MAX = 4096;           // offsets whose table is read from LDS (16 KB beside the tiles)

// before the large kernels: workgroups [0, eb) form e[h][o] = log2 units of the head's bias at offset o, 256 / 8 offsets x 8 heads at a time; the others (backward)
// delta[b][h][q] = dout . out, 16 lanes a row.  Both go on by their number of workgroups, at most MAX_WG
template <typename T>
__global__ __launch_bounds__(256) void rel_pre_kernel(RelP p, float* e, int eb) {
    if ((int)blockIdx.x < eb) {
        for (int o = blockIdx.x * 32 + (threadIdx.x & 31); o < p.nd; o += eb * 32) {
            const int c = p.buckets ? p.buckets[o] : o;
            for (int h = threadIdx.x >> 5; h < p.H; h += 8) e[(long)h * p.nd + o] = rel_log2_bias(p.table, p.tdt, c, p.nb, h, p.H);
        }
        return;
    }
    const T *o = static_cast<const T*>(p.o), *dout = static_cast<const T*>(p.dout);
    const int Nq = p.Nq, H = p.H, D = p.D;
    const long rows = (long)p.B * Nq * H;
    const int c = (threadIdx.x & 15) * 8;
    for (long row = (long)(blockIdx.x - eb) * 16 + (threadIdx.x >> 4); row < rows; row += (long)(gridDim.x - eb) * 16) {             // (b Nq + q) H + h
        float s = 0.f;
        if (c < D) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f32x4 a = load4(o + row * D + c + 4 * u), g = load4(dout + row * D + c + 4 * u);
#pragma unroll
                for (int j = 0; j < 4; ++j) s = __builtin_fmaf(a[j], g[j], s);
            }
        }
        s = group16_sum(s);
        if ((threadIdx.x & 15) == 0) {
            const long bq = row / H;
            p.delta[((bq / Nq) * H + row % H) * Nq + bq % Nq] = s;
        }
    }
}

// merge of the split forward: 32 lanes a row, 4 columns a lane
template <typename T>
__global__ __launch_bounds__(256) void rel_combine_kernel(RelP p) {
    const long rows = (long)p.B * p.H * p.Nq, row = (long)blockIdx.x * 8 + threadIdx.x / 32;       // (b H + h) Nq + q
    const int d = (threadIdx.x & 31) * 4;
    if (row >= rows) return;
    float M = -INFINITY;
    for (int s = 0; s < p.nsplit; ++s) M = fmaxf(M, p.pm[s * rows + row]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.nsplit; ++s) {
        const float w = __builtin_amdgcn_exp2f(p.pm[s * rows + row] - ref);          // an empty split: exp2(-inf) = 0
        L = __builtin_fmaf(w, p.pl[s * rows + row], L);
        if (d < p.D) {
            const f32x4 v = load4(p.po + (s * rows + row) * p.D + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = __builtin_fmaf(w, v[j], a[j]);
        }
    }
    const float f = L == 0.f ? 0.f : 1.f / L;
    const long bh = row / p.Nq, q = row % p.Nq, b = bh / p.H, h = bh % p.H;
    if (d < p.D) store4(static_cast<T*>(p.out) + ((b * p.Nq + q) * p.H + h) * p.D + d, (f32x4){a[0] * f, a[1] * f, a[2] * f, a[3] * f});
    if (d == 0 && p.lse) p.lse[row] = L == 0.f ? INFINITY : M + __builtin_amdgcn_logf(L);
}

// ... of many splits (few rows): a workgroup a row, 32 groups of 32 lanes take every 32nd split, joined in order
template <typename T>
__global__ __launch_bounds__(1024) void rel_combine_row_kernel(RelP p) {
    __shared__ float red[32][32 * 4 + 4];
    const long rows = (long)p.B * p.H * p.Nq, row = blockIdx.x;
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, d = lane * 4;
    float M = -INFINITY;
    for (int s = lane; s < p.nsplit; s += 32) M = fmaxf(M, p.pm[s * rows + row]);
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = g; s < p.nsplit; s += 32) {
        const float w = __builtin_amdgcn_exp2f(p.pm[s * rows + row] - ref);
        L = __builtin_fmaf(w, p.pl[s * rows + row], L);
        if (d < p.D) {
            const f32x4 v = load4(p.po + (s * rows + row) * p.D + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = __builtin_fmaf(w, v[j], a[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[g][d + j] = a[j];
    if (lane == 0) red[g][128] = L;
    __syncthreads();
    if (g) return;
    L = 0.f;
    a = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        L += red[i][128];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] += red[i][d + j];
    }
    const float f = L == 0.f ? 0.f : 1.f / L;
    const long bh = row / p.Nq, q = row % p.Nq, b = bh / p.H, h = bh % p.H;
    if (d < p.D) store4(static_cast<T*>(p.out) + ((b * p.Nq + q) * p.H + h) * p.D + d, (f32x4){a[0] * f, a[1] * f, a[2] * f, a[3] * f});
    if (d == 0 && p.lse) p.lse[row] = L == 0.f ? INFINITY : M + __builtin_amdgcn_logf(L);
}

// sum of the n parts of dQ, or of dK and dV (grid y), in their order: 32 lanes a row, 4 columns a lane.  Nq > 0: rows (b H + h) Nq + q, and delta takes its correction, the
// sum of pm; else rows as in out and out2 (unscaled)
template <typename T>
__global__ __launch_bounds__(256) void rel_join_kernel(const float* part, int n, long rows, int D, float scale, T* out, T* out2, int Nq, int H, const float* pm, float* delta) {
    if (blockIdx.y) { part += n * rows * D; out = out2; scale = 1.f; }
    const long row = (long)blockIdx.x * 8 + threadIdx.x / 32;
    const int d = (threadIdx.x & 31) * 4;
    if (row >= rows) return;
    if (d < D) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < n; ++s) a += load4(part + (s * rows + row) * D + d);
        long to = row;
        if (Nq) {
            const long bh = row / Nq, q = row % Nq, b = bh / H, h = bh % H;
            to = (b * Nq + q) * H + h;
        }
        store4(out + to * D + d, (f32x4){a[0] * scale, a[1] * scale, a[2] * scale, a[3] * scale});
    }
    if (Nq && d == 0) {
        float off = 0.f;
        for (int s = 0; s < n; ++s) off += pm[s * rows + row];
        delta[row] += off;
    }
}

// G[h][o]: sums by offset of the partials, 64 offsets x 16 runs of partials a workgroup, joined in order; written as the table's gradient at once where every offset is
// its own bucket (dt).
//   LINE: slab rows (b, key tile, part of the queries) of len places: row t of the part that begins at query q holds offset o at place
//         o - (gw - 1) - q_start + 32 + 32 t - q
//   DENSE: M[z][h][a][c]: the pairs of a query cell a and the key cell = its cell - offset, where both lie on the grid
//   FEW:   the same, of tokens on few cells of a large grid: only the cells that hold a query whose key cell holds a key are walked (most offsets have none)
struct FoldP { const float* slab; float* G; void* dt; long len; int tdt, B, H, nd, tiles, base; int gd, gh, gw, vol, q0, QC, KC, ld, parts, ksplit, klog, nqb, blk; };
enum { FOLD_LINE = 0, FOLD_DENSE = 1, FOLD_FEW = 2 };
template <int MODE>
__global__ __launch_bounds__(1024) void rel_fold_kernel(FoldP f) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, run = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y;
    const int o0 = (blockIdx.z * gridDim.x + blockIdx.x) * 64, o = o0 + lane;                   // (z: past MAX_WG workgroups)
    if (o0 >= f.nd) return;
    float s = 0.f;
    if constexpr (MODE == FOLD_LINE) {
        // the key tiles that may hold one of the workgroup's offsets, W of them from ta on, for every batch entry and part
        const bool any = o0 + 63 >= f.base - 32 * f.tiles && o0 <= f.base + f.nqb * f.blk;           // (a line may be far longer than the tokens on it)
        const int W = (int)(f.len / 32) + 3, n = any ? f.B * f.ksplit * W : 0, i0 = (int)((long)n * run / 16), i1 = (int)((long)n * (run + 1) / 16);
        int bp = i0 / W, j = i0 - bp * W;
// (loads unconditional, eight in flight: a load under a condition is waited for before the next one)
#pragma unroll 8
        for (int i = i0; i < i1; ++i) {
            const int part = bp & (f.ksplit - 1), b = bp >> f.klog;
            const int q0 = (int)((unsigned)(part * f.nqb) >> f.klog), q1 = (int)((unsigned)((part + 1) * f.nqb) >> f.klog);       // (in blocks)
            const int from = f.base - 32 + q0 * f.blk, ta = (from - o0 - 63 + 31) >> 5, t = ta + j, u = o - from + 32 * t;
            const bool in = (unsigned)t < (unsigned)f.tiles && (unsigned)u < (unsigned)((q1 - q0) * f.blk + 32);
            const float v = f.slab[in ? ((((long)b * f.H + h) * f.tiles + t) * f.ksplit + part) * f.len + u : 0];
            s += in ? v : 0.f;
            if (++j == W) { j = 0; ++bp; }
        }
    } else {
        const int sx = 2 * f.gw - 1, sy = 2 * f.gh - 1;
        const int dx = o % sx - (f.gw - 1), dy = o / sx % sy - (f.gh - 1), dz = o / sx / sy - (f.gd - 1);
        const int shift = (dz * f.gh + dy) * f.gw + dx, first = f.q0 % f.vol;              // the query's cell counts from q_start (the raster may begin inside the grid)
        const long part = (long)f.H * f.QC * f.ld;
        const float* m = f.slab + (long)h * f.QC * f.ld;
        if constexpr (MODE == FOLD_FEW) {
            for (int seg = 0; seg < 2; ++seg) {                                              // the queries' cells [first, ..) and, where they go round, [0, ..)
                const int lo = max(seg ? 0 : first, max(0, shift)), hi = min(seg ? first + f.QC - f.vol : min(first + f.QC, f.vol), min(f.vol, f.KC + shift));
                for (int cell = lo + run; __any(cell < hi && o < f.nd); cell += 16) {
                    const int r = cell / f.gw, x = cell - r * f.gw, z = r / f.gh, y = r - z * f.gh, a = cell - first + (seg ? f.vol : 0);
                    if (cell >= hi || o >= f.nd || (unsigned)(x - dx) >= (unsigned)f.gw || (unsigned)(y - dy) >= (unsigned)f.gh || (unsigned)(z - dz) >= (unsigned)f.gd) continue;
                    for (int i = 0; i < f.parts; ++i) s += m[i * part + (long)a * f.ld + cell - shift];
                }
            }
        } else {
            // units of 8 cells along x of the rows (z, y) that have a partner
            const int nz = f.gd - abs(dz), ny = f.gh - abs(dy), z0 = max(0, dz), y0 = max(0, dy), XC = (f.gw + 7) / 8;
            const int n = o < f.nd ? nz * ny * XC : 0;
            for (int z = 0; z < f.parts; ++z, m += part)
                for (int u = run; __any(u < n); u += 16) {
                    const int row = u / XC, x8 = (u - row * XC) * 8, rz = row / ny, ry = row - rz * ny, cell = ((z0 + rz) * f.gh + y0 + ry) * f.gw + x8;
                    float v[8];
                    bool in[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int x = x8 + i, c = cell + i - shift;
                        int a = cell + i - first;
                        a = a < 0 ? a + f.vol : a;
                        in[i] = u < n && x < f.gw && (unsigned)(x - dx) < (unsigned)f.gw && a < f.QC && c < f.KC;
                        v[i] = m[in[i] ? (long)a * f.ld + c : 0];
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) s += in[i] ? v[i] : 0.f;
                }
        }
    }
    red[run][lane] = s;
    __syncthreads();
    if (run == 0 && o < f.nd) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += red[i][lane];
        if (f.dt) {
            if (f.tdt == PASSION_BF16) static_cast<bf16_t*>(f.dt)[(long)o * f.H + h] = (bf16_t)s;
            else static_cast<float*>(f.dt)[(long)o * f.H + h] = s;
        } else f.G[(long)h * f.nd + o] = s;
    }
}

// a grid smaller than a tile: out[h][a][c] = sum of M over its parts and over the copies of cells a < qc, c < kc.  A workgroup a pair, in a fixed order
__global__ __launch_bounds__(256) void rel_copies_kernel(RelP p, int ld, int qc, int kc, float* out) {
    __shared__ float red[4];
    const int a0 = blockIdx.x / kc, c0 = blockIdx.x % kc, h = blockIdx.y;
    const int ma = (p.QC - a0 + p.vol - 1) / p.vol, mc = (p.KC - c0 + p.vol - 1) / p.vol, n = p.parts * ma * mc;
    float s = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 256) {
        const int c = i % mc, a = i / mc % ma, z = i / mc / ma;
        s += p.slab[(((long)z * p.H + h) * p.QC + a0 + a * p.vol) * ld + c0 + c * p.vol];
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) out[((long)h * qc + a0) * kc + c0] = (red[0] + red[1]) + (red[2] + red[3]);
}

// dtable[c][h] = sum of G[h][o] over the offsets of bucket c, in their order.  Few buckets: a workgroup a bucket; many: a thread a bucket, the map through LDS, four offsets a read
// (an offset at a time waited for each read: 52 ns an offset)
template <typename TT>
__global__ __launch_bounds__(256) void rel_bucket_few_kernel(const float* G, const int* buckets, TT* dt, int nd, int H) {
    __shared__ float red[4];
    const int c = blockIdx.x, h = blockIdx.y;
    float s = 0.f;
#pragma unroll 8
    for (int o = threadIdx.x; o < nd; o += 256) {
        const float v = G[(long)h * nd + o];
        s += buckets[o] == c ? v : 0.f;
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) dt[(long)c * H + h] = from_f32<TT>((red[0] + red[1]) + (red[2] + red[3]));
}
template <typename TT>
__global__ __launch_bounds__(256) void rel_bucket_many_kernel(const float* G, const int* buckets, TT* dt, int nd, int nb, int H) {
    __shared__ __attribute__((aligned(16))) int bk[1024];
    __shared__ __attribute__((aligned(16))) float gv[1024];
    const int c = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
    float s = 0.f;
    for (int o0 = 0; o0 < nd; o0 += 1024) {
        __syncthreads();
        for (int i = threadIdx.x; i < 1024; i += 256) {
            bk[i] = o0 + i < nd ? buckets[o0 + i] : -1;
            gv[i] = o0 + i < nd ? G[(long)h * nd + o0 + i] : 0.f;
        }
        __syncthreads();
#pragma unroll 4
        for (int i = 0; i < 1024; i += 4) {
            const int4 b = *reinterpret_cast<const int4*>(bk + i);
            const f32x4 g = *reinterpret_cast<const f32x4*>(gv + i);
            s += b.x == c ? g[0] : 0.f;
            s += b.y == c ? g[1] : 0.f;
            s += b.z == c ? g[2] : 0.f;
            s += b.w == c ? g[3] : 0.f;
        }
    }
    if (c < nb) dt[(long)c * H + h] = from_f32<TT>(s);
}

int blk_of(int dtype) { return dtype == PASSION_BF16 ? 64 : 32; }
long tiles32(long n) { return (n + 31) / 32; }

// which way to the bias: a 1D raster without wrap-around by windows, a small box of offsets from LDS, else from memory.  Forward + backward, 8 heads of 64, from LDS / from memory:
// 4 x 2048^2 over 8^3 cells 370 / 397 us (forward alone 71 / 82), 2 x 2000^2 of 32 over 5^3 280 / 352, f32 2048^2 547 / 570; 2 x 512^2 over 8^3 97 / 95.  Tables over 16 KB cost a
// workgroup a CU: 9^3 cells 138 / 137 (heads of 128: 236 / 211), 12^3 592 / 396
int bias_mode(const RelP& p) {
    if (!p.table) return 0;
    if (p.gd == 1 && p.gh == 1 && p.Nk <= p.gw && (long)p.q0 + p.Nq <= p.gw) return 2;
    return p.nd <= BOX_MAX ? 1 : 3;
}
// few query rows: all heads of a key / value head in one tile, the bias read straight from the table.  Against the ordinary way (expansion of all offsets first), whole call, bf16:
// 4 x 1 x 6000 tokens, 8 heads of 64 on 2: 14.9 / 19.9 us (f32 26.5 / 33.2), 1 x 16 x 6000 14.2 / 17.8.  Not better where heads share nothing and workgroups are many: 16 x 1 x 1000,
// 8 heads on 8, 30 / 24 us, f32 1 x 16 x 6000 27 / 23
bool few_rows(const RelP& p) { return (long)p.Nq * (p.H / p.Hkv) <= 32 && p.Nq <= 16; }

// tokens on few of the grid's cells: the sums by offset walk the tokens' cells and not the grid's.  8 heads, the grid's cells / the tokens': 200 tokens on 64^3 cells 510 ms /
// 0.92 ms (and times 64 with every doubling of the sides), 300 or 500 on 16^3 190 us / 27 to 43 us, 120 on 10^3 33 / 9 us
bool few_cells(int QC, int KC, int vol) { return 8 * hmin(QC, KC) < vol; }

// the forward's key ranges.  Few rows: a block of keys a workgroup up to 2048 of them (all of a short cache in flight at once: 4 x 1 x 6000 14.9 us, up to 512 of them 16.7; a long cache pays
// for the join: 1 x 1 x 60000 51 and 31 us); else until there is a wavefront on three of four SIMDs, two blocks each at least: 128 x 2048, 8 heads of 64, whole / in parts 73 / 23 us,
// 1000^2 40 / 21 (41 with a limit of 256 wavefronts, 29 with one of 2048), 64 x 8000 276 / 21
int pick_split(const RelP& p, int dtype) {
    const long tiles = (p.pack ? tiles32((long)p.Nq * (p.H / p.Hkv)) * p.Hkv : tiles32(p.Nq) * p.H) * p.B;
    const int nblk = (p.Nk + blk_of(dtype) - 1) / blk_of(dtype);
    if (p.few) return (int)hmax(1, hmin(nblk, 2048 / tiles));
    int s = 1;
    while (tiles * s < 768 && nblk / (2 * s) >= 2) s *= 2;
    return s;
}
// the backward's: parts (a power of two) of at least 128 of the n tokens that a wavefront walks, until there is a wavefront on three of four SIMDs.
// Forward + backward, us, whole / in parts: 185 x 1626 tokens, 2 heads of 128, f32 555 / 220; 2 x 2774^2, 2 heads of 64 on one, f32 1495 / 571; 2258^2, 2 heads of 128 on
// one, bf16 779 / 165; 2048^2 over 8^3 cells, 8 heads of 64, bf16 241 / 187.  Up to a wavefront on every SIMD the last is as fast, the second takes 647
int pick_split_bwd(long tiles, int n) {
    int s = 1;
    while (tiles * s < 768 && n / (2 * s) >= 128) s *= 2;
    return s;
}
// wavefronts a workgroup, which share the staged tiles: forward + backward over a line, 8 heads of 64, bf16, by one / two / four: 512^2 74 / 59 / 57 us, 1024^2 143 / 93 / 80, 4 x 1024^2
// 365 / 163 / 131 (f32 675 / 501 / 431); the limits are those of one workgroup a CU, and below them two are the choice, though four are faster there too (3 x 1024^2, 768 wavefronts: 160 / 127).  Key-major with heads over 64 wide: LDS and registers hold one workgroup a CU,
// and a workgroup more than there are CUs is a second round: four as soon as two would begin one (1077^2, 8 heads of 96 on 2, f32, 544 wavefronts: forward + backward 804 us by two, 481 by four)
int pick_waves(long rows32, long others, bool alone = false) {
    const long waves = rows32 * others;
    return rows32 >= 4 && waves > (alone ? 512 : 899) ? 4 : rows32 >= 2 && waves > (alone ? 256 : 383) ? 2 : 1;
}

int setup(RelP& p, int dtype, int B, int Nq, int Nk, int H, int Hkv, int D, int gd, int gh, int gw, int q_start, const void* table, int tdt, const int* buckets, int nb,
          const uint8_t* mask, float scale) {
    if ((dtype != PASSION_F32 && dtype != PASSION_BF16) || B < 1 || B > 65535 || Nq < 1 || Nk < 1 || H < 1 || Hkv < 1 || H % Hkv || H > 65535) return -1003;
    if (D < 8 || D > 128 || D % 8) return -1003;
    if (Nq > (1 << 30) || Nk > (1 << 30) || q_start < 0 || q_start > (1 << 30)) return -1003;
    if (table) {
        if (gd < 1 || gh < 1 || gw < 1 || (tdt != PASSION_F32 && tdt != PASSION_BF16) || nb < 1) return -1003;
        const int64_t a = 2LL * gd - 1, b = 2LL * gh - 1, c = 2LL * gw - 1;
        if (a > (1 << 30) || b > (1 << 30) || c > (1LL << 31) || a * b > (1 << 30) || a * b * c > (1LL << 30)) return -1003;
        p.gd = gd; p.gh = gh; p.gw = gw; p.vol = (int)((int64_t)gd * gh * gw); p.nd = (int)(a * b * c);
        p.omax = ((gd - 1) * (2 * gh - 1) + gh - 1) * (2 * gw - 1) + gw - 1;
        if (!buckets && nb != p.nd) return -1003;
        p.table = table; p.buckets = buckets; p.nb = nb; p.tdt = tdt;
    }
    p.B = B; p.Nq = Nq; p.Nk = Nk; p.H = H; p.Hkv = Hkv; p.D = D; p.q0 = q_start; p.mask = mask;
    p.scale = scale; p.c = scale * 1.4426950408889634f;
    p.nsplit = p.ksplit = 1;
    p.bias = bias_mode(p);
    return 0;
}

// partials of the table's gradient, in floats; sets what the kernels need to know of them
long slab_floats(RelP& p, int dtype) {
    const long blk = blk_of(dtype);
    if (p.bias == 2) {
        const long nqb = (p.Nq + blk - 1) / blk;
        p.slab_len = (nqb + p.ksplit - 1) / p.ksplit * blk + 32;
        return (long)p.B * p.H * tiles32(p.Nk) * p.ksplit * p.slab_len;
    }
    p.QC = (int)hmin(p.Nq, p.vol * hmax(1, 128 / p.vol)); p.KC = (int)hmin(p.Nk, p.vol * hmax(1, 64 / p.vol));
    const long passes = (long)p.B * ((p.Nq + p.QC - 1) / p.QC) * ((p.Nk + p.KC - 1) / p.KC), nkb = (p.KC + blk - 1) / blk, waves = tiles32(p.QC) * nkb * p.H;
    p.parts = (int)hmax(1, hmin(passes, 2048 / waves));            // about two wavefronts a SIMD
    return (long)p.parts * p.H * p.QC * nkb * blk;
}

// more than 256 buckets: the last sum reads every offset for every 256 of them: 11.5 ns an offset (2 10^6 offsets, 10^4 to 10^5 buckets: 24 ms in all; 52 ns by one offset a read: 106 ms), and
// 1.4 10^13 pairs of offset and bucket a second where they fill the card.  Past 2^46 pairs, seconds, the gradient is refused
bool too_many_pairs(const RelP& p) { return p.buckets && p.nb > 256 && (double)p.nd * (double)hmax((long)p.nb * p.H, 1L << 19) > (double)(1L << 46); }

int run(const RelP& p, int dtype, int what, int nw, hipStream_t st) { return dtype == PASSION_BF16 ? rel_run_bf16(p, what, nw, st) : rel_run_f32(p, what, nw, st); }

// layout of the workspaces, in floats
struct Ws { long e, po, pm, pl, delta, slab, cells, G, total; };
Ws fwd_ws(RelP& p, int dtype) {
    p.few = few_rows(p);
    p.pack = p.few && p.H > p.Hkv;
    if (p.bias == 1 && p.few) p.bias = 3;
    p.nsplit = pick_split(p, dtype);
    const long rows = (long)p.B * p.H * p.Nq;
    Ws w{};
    long at = 0;
    auto take = [&](long n) { const long r = at; at += (n + 63) / 64 * 64; return r; };
    w.e = take(p.bias && !p.few ? (long)p.H * p.nd : 0);
    w.po = take(p.nsplit > 1 ? p.nsplit * rows * p.D : 0);
    w.pm = take(p.nsplit > 1 ? p.nsplit * rows : 0);
    w.pl = take(p.nsplit > 1 ? p.nsplit * rows : 0);
    w.total = at;
    return w;
}
Ws bwd_ws(RelP& p, int dtype, bool want_table) {
    Ws w{};
    long at = 0;
    auto take = [&](long n) { const long r = at; at += (n + 63) / 64 * 64; return r; };
    w.e = take(p.bias ? (long)p.H * p.nd : 0);
    w.delta = take((long)p.B * p.H * p.Nq);
    p.nsplit = pick_split_bwd(tiles32(p.Nq) * p.H * p.B, p.Nk);
    p.ksplit = pick_split_bwd(tiles32(p.Nk) * p.Hkv * p.B, p.Nq);
    while ((long)p.ksplit * ((p.Nq + 31) / 32) > (1 << 30)) p.ksplit /= 2;            // (rel_fold_kernel multiplies parts by blocks in 32 bits)
    const long rows = (long)p.B * p.H * p.Nq, krows = (long)p.B * p.Nk * p.Hkv;
    w.po = take(hmax(p.nsplit > 1 ? p.nsplit * rows * p.D : 0, p.ksplit > 1 ? 2 * p.ksplit * krows * p.D : 0));       // dQ's parts, then those of dK and dV
    w.pm = take(p.nsplit > 1 ? p.nsplit * rows : 0);
    if (p.bias && want_table) {
        w.slab = take(slab_floats(p, dtype));
        w.cells = take(p.bias != 2 && hmax(p.QC, p.KC) > p.vol ? p.H * hmin(p.QC, p.vol) * hmin(p.KC, p.vol) : 0);
        w.G = take(p.buckets ? (long)p.H * p.nd : 0);
    }
    w.total = at;
    return w;
}
int pre(RelP& p, int dtype, float* e, hipStream_t st) {
    const int eb = e ? (int)hmin((p.nd + 31) / 32, MAX_WG) : 0;
    const long db = p.delta ? hmin(((long)p.B * p.Nq * p.H + 15) / 16, MAX_WG) : 0;
    if (dtype == PASSION_BF16) hipLaunchKernelGGL(rel_pre_kernel<bf16_t>, dim3((unsigned)(eb + db)), dim3(256), 0, st, p, e, eb);
    else hipLaunchKernelGGL(rel_pre_kernel<float>, dim3((unsigned)(eb + db)), dim3(256), 0, st, p, e, eb);
    LAUNCH_RET();
    p.e = e;
    return 0;
}
int join(int dtype, const float* part, int n, long rows, int D, float scale, void* out, void* out2, int Nq, int H, const float* pm, float* delta, hipStream_t st) {
    const dim3 grid((unsigned)((rows + 7) / 8), out2 ? 2 : 1);
    if (dtype == PASSION_BF16) hipLaunchKernelGGL(rel_join_kernel<bf16_t>, grid, dim3(256), 0, st, part, n, rows, D, scale, static_cast<bf16_t*>(out), static_cast<bf16_t*>(out2), Nq, H, pm, delta);
    else hipLaunchKernelGGL(rel_join_kernel<float>, grid, dim3(256), 0, st, part, n, rows, D, scale, static_cast<float*>(out), static_cast<float*>(out2), Nq, H, pm, delta);
    LAUNCH_RET();
    return 0;
}
bool misaligned(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; }
int strides(RelP& p, int dtype, const int64_t* sq, const int64_t* sk, const int64_t* sv) {
    const int unit = dtype == PASSION_BF16 ? 8 : 4;
    for (int i = 0; i < 3; ++i) {                                                 // (the stride of a dimension of one may be anything)
        p.qs[i] = (i == 0 ? p.B : i == 1 ? p.Nq : p.H) > 1 ? sq[i] : 0;
        p.ks[i] = (i == 0 ? p.B : i == 1 ? p.Nk : p.Hkv) > 1 ? sk[i] : 0;
        p.vs[i] = (i == 0 ? p.B : i == 1 ? p.Nk : p.Hkv) > 1 ? sv[i] : 0;
        if (p.qs[i] % unit || p.ks[i] % unit || p.vs[i] % unit) return -1005;
    }
    for (const int64_t s : {(int64_t)p.qs[1], (int64_t)p.ks[1], (int64_t)p.vs[1], (int64_t)p.H * p.D})           // 32-bit lane offsets over a block of 64 tokens
        if (s < 0 || s >= (1 << 23)) return -1005;
    return 0;
}

}  // namespace

extern "C" int64_t passion_rel_attn_workspace_floats(int dtype, int backward, int B, int Nq, int Nk, int H, int Hkv, int D, int gd, int gh, int gw, int q_start,
                                                     int has_table, int has_buckets, int nb) {
    RelP p{};
    static const int dummy = 0;
    const int rc = setup(p, dtype, B, Nq, Nk, H, Hkv, D, gd, gh, gw, q_start, has_table ? &dummy : nullptr, PASSION_F32, has_buckets ? &dummy : nullptr, nb, nullptr, 1.f);
    if (rc) return rc;
    if (backward == 1 && too_many_pairs(p)) return -1003;
    return backward ? bwd_ws(p, dtype, backward == 1).total : fwd_ws(p, dtype).total;
}

extern "C" int passion_rel_attn_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int dtype, int B,
                                    int Nq, int Nk, int H, int Hkv, int D, int gd, int gh, int gw, int q_start, const void* table, int table_dtype, const int* buckets,
                                    int nb, const uint8_t* mask, float scale, void* out, float* lse, float* workspace, void* stream) {
    RelP p{};
    int rc = setup(p, dtype, B, Nq, Nk, H, Hkv, D, gd, gh, gw, q_start, table, table_dtype, buckets, nb, mask, scale);
    if (rc) return rc;
    if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides) return -1003;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || (workspace && misaligned(workspace))) return -1005;
    if ((rc = strides(p, dtype, q_strides, k_strides, v_strides))) return rc;
    p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse;
    hipStream_t st = (hipStream_t)stream;
    const Ws w = fwd_ws(p, dtype);
    if (w.total && !workspace) return -1003;
    if (p.bias && !p.few && (rc = pre(p, dtype, workspace + w.e, st))) return rc;
    p.po = workspace + w.po; p.pm = workspace + w.pm; p.pl = workspace + w.pl;
    const long rows32 = p.pack ? tiles32((long)p.Nq * (p.H / p.Hkv)) : tiles32(p.Nq);
    if ((rc = run(p, dtype, 0, pick_waves(rows32, (long)(p.pack ? p.Hkv : p.H) * p.B * p.nsplit), st))) return rc;
    if (p.nsplit > 1) {
        const long rows = (long)p.B * p.H * p.Nq;
        if (p.nsplit > 16) {
            if (dtype == PASSION_BF16) hipLaunchKernelGGL(rel_combine_row_kernel<bf16_t>, dim3((unsigned)rows), dim3(1024), 0, st, p);
            else hipLaunchKernelGGL(rel_combine_row_kernel<float>, dim3((unsigned)rows), dim3(1024), 0, st, p);
        } else if (dtype == PASSION_BF16) hipLaunchKernelGGL(rel_combine_kernel<bf16_t>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p);
        else hipLaunchKernelGGL(rel_combine_kernel<float>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p);
        LAUNCH_RET();
    }
    return 0;
}

extern "C" int passion_rel_attn_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int dtype, int B,
                                    int Nq, int Nk, int H, int Hkv, int D, int gd, int gh, int gw, int q_start, const void* table, int table_dtype, const int* buckets,
                                    int nb, const uint8_t* mask, float scale, const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv, void* dtable,
                                    float* workspace, void* stream) {
    RelP p{};
    int rc = setup(p, dtype, B, Nq, Nk, H, Hkv, D, gd, gh, gw, q_start, table, table_dtype, buckets, nb, mask, scale);
    if (rc) return rc;
    if (!q || !k || !v || !out || !dout || !lse || !dq || !dk || !dv || !workspace || !q_strides || !k_strides || !v_strides || (dtable && (!table || too_many_pairs(p)))) return -1003;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(dout) || misaligned(dq) || misaligned(dk) || misaligned(dv) || misaligned(workspace))
        return -1005;
    if ((rc = strides(p, dtype, q_strides, k_strides, v_strides))) return rc;
    p.q = q; p.k = k; p.v = v; p.o = out; p.dout = dout; p.lse = const_cast<float*>(lse); p.dq = dq; p.dk = dk; p.dv = dv;
    hipStream_t st = (hipStream_t)stream;
    const Ws w = bwd_ws(p, dtype, dtable != nullptr);
    p.delta = workspace + w.delta;
    if ((rc = pre(p, dtype, p.bias ? workspace + w.e : nullptr, st))) return rc;
    p.slab = dtable ? workspace + w.slab : nullptr;
    p.po = workspace + w.po;
    p.pm = workspace + w.pm;
    if ((rc = run(p, dtype, 1, pick_waves(tiles32(Nq), (long)H * B * p.nsplit), st))) return rc;
    const long rows = (long)B * H * Nq, krows = (long)B * Nk * Hkv;
    if (p.nsplit > 1 && (rc = join(dtype, p.po, p.nsplit, rows, D, scale, dq, nullptr, Nq, H, p.pm, p.delta, st))) return rc;
    if ((rc = run(p, dtype, 2, pick_waves(tiles32(Nk), (long)Hkv * B * p.ksplit, D > 64), st))) return rc;
    if (p.ksplit > 1 && (rc = join(dtype, p.po, p.ksplit, krows, D, scale, dk, dv, 0, 0, nullptr, nullptr, st))) return rc;
    if (dtable) {
        const long nkb = p.bias == 2 ? 0 : (p.KC + blk_of(dtype) - 1) / blk_of(dtype);
        if (p.bias != 2 && (rc = run(p, dtype, 3, pick_waves(tiles32(p.QC), nkb * H * p.parts), st))) return rc;
        float* G = workspace + w.G;
        FoldP f{p.slab, G, buckets ? nullptr : dtable, p.slab_len, table_dtype, B, H, p.nd, (int)tiles32(Nk), p.gw - 1 + p.q0, p.gd, p.gh, p.gw, p.vol, p.q0, p.QC, p.KC,
                (int)(nkb * blk_of(dtype)), p.parts, p.ksplit, __builtin_ctz(p.ksplit), (Nq + blk_of(dtype) - 1) / blk_of(dtype), blk_of(dtype)};
        if (p.bias != 2 && hmax(p.QC, p.KC) > p.vol) {
            f.QC = (int)hmin(p.QC, p.vol);
            f.KC = (int)hmin(p.KC, p.vol);
            hipLaunchKernelGGL(rel_copies_kernel, dim3(f.QC * f.KC, H), dim3(256), 0, st, p, f.ld, f.QC, f.KC, workspace + w.cells);
            LAUNCH_RET();
            f.slab = workspace + w.cells;
            f.ld = f.KC;
            f.parts = 1;
        }
        const int groups = (p.nd + 63) / 64, wide = (int)hmin(groups, MAX_WG);
        const dim3 wgs(wide, H, (groups + wide - 1) / wide);
        if (p.bias == 2) hipLaunchKernelGGL(rel_fold_kernel<FOLD_LINE>, wgs, dim3(1024), 0, st, f);
        else if (few_cells(f.QC, f.KC, f.vol)) hipLaunchKernelGGL(rel_fold_kernel<FOLD_FEW>, wgs, dim3(1024), 0, st, f);
        else hipLaunchKernelGGL(rel_fold_kernel<FOLD_DENSE>, wgs, dim3(1024), 0, st, f);
        LAUNCH_RET();
        if (buckets) {
            const bool few = nb <= 256;
            if (table_dtype == PASSION_BF16) {
                if (few) hipLaunchKernelGGL(rel_bucket_few_kernel<bf16_t>, dim3(nb, H), dim3(256), 0, st, G, buckets, (bf16_t*)dtable, p.nd, H);
                else hipLaunchKernelGGL(rel_bucket_many_kernel<bf16_t>, dim3((nb + 255) / 256, H), dim3(256), 0, st, G, buckets, (bf16_t*)dtable, p.nd, nb, H);
            } else {
                if (few) hipLaunchKernelGGL(rel_bucket_few_kernel<float>, dim3(nb, H), dim3(256), 0, st, G, buckets, (float*)dtable, p.nd, H);
                else hipLaunchKernelGGL(rel_bucket_many_kernel<float>, dim3((nb + 255) / 256, H), dim3(256), 0, st, G, buckets, (float*)dtable, p.nd, nb, H);
            }
            LAUNCH_RET();
        }
    }
    return 0;
}
