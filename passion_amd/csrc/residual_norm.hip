// The residual step between two transformer blocks, one launch each way:
//     u = post(h),   r = x + scale * gate * u,   y = pre(r)
// h: a block's output, x: the residual stream, post / pre: LayerNorm or RMSNorm over the C channels (each optional), gate: per sample
// and channel or per token and channel, scale: per channel.  The glue of the reference's Transformer (code/models/mmformer.py:230-256,
// 284-300: x + dropout(f(norm(x))), norm of the next block) in the form a gated, post-normed block has it.
//
// Bound by memory: forward reads x, h (, a token gate) and writes r, y once; backward reads x, h, dr, dy and writes dx, dh.  The backward
// forms r again from x and h instead of reading it: the same bytes, and the parameter gradients see the unrounded r.
//
// Layout: a row = C channels over TPR threads (a power of two, 8 channels a thread: one 16-byte access a thread and bf16 tensor), 256 / TPR
// rows a workgroup (one row from TPR = 256 on).  Rows of up to 512 channels live inside one wavefront: moments by butterfly shuffles.
// Wider ones exchange (sum, second moment about the wavefront's own mean) through LDS and join them in wavefront order -- one barrier
// a norm and no cancellation in the variance.  Channel vectors (weights, scale, a sample's gate) stay in registers over a workgroup's rows.
// Column sums of the backward: in registers over the workgroup's rows (of one sample), one partial per workgroup, folded in
// workgroup order by a second kernel: no atomics, results repeat bit for bit.
// All arithmetic and every sum is f32; x, h, y, r and the gradients round once when they are stored.
// 8 x 4096 x 2048 bf16 with a sample's gate: forward 117 us (4.6 TB/s), backward 180 (4.5 TB/s; two wavefronts a SIMD with one row of each in flight), fold of the column sums 13.
// 3 x 4001 x 765 f32 with a token's gate: 38 + 68 + 9 us; rows of an odd width are read and written 4 bytes a thread.
// Rows of more than 4096 channels: 1024 threads have 128 registers each, the backward wants about 230 and spills 210 to 254 (odd widths 417 to 538; their forward 287): 67 million elements
// bf16 forward / backward at 4096 wide 207 / 201 us, 8192 wide 209 / 1657, 4104 wide 295 / 2783, 6001 wide 1127 / 2694.
#include "common.h"
#include "passion_hip.h"

namespace {

constexpr int RN_MAX_C = 8192, VPT = 8;
// rows a sample: the kernels count them in 32 bits, and a workgroup's last step passes the end by less than its chunk (below 2^27 rows of anything that memory holds).
// (Counted from the workgroup's own first row, 12003 x 765 took 127 us instead of 123; unsigned, 131)
constexpr int RN_MAX_N = 0x7fffffff - (1 << 27);

struct RnP {
    const void *x, *h, *gate;                 // [B][N][C]; gate [B][C] or [B][N][C]
    const float *w1, *b1, *w2, *b2, *scale;   // post, pre (f32 [C]) and the residual scale; NULL: 1 / 0
    void *r, *y;
    float* stat;                              // [B N][4]: mean, rstd of post; mean, rstd of pre
    const void *dr, *dy;                      // backward; NULL: zero
    void *dx, *dh, *dgate_tok;
    float* part;                              // [blocks][6][C]: dw1, db1, dw2, db2, dscale, dgate of the sample
    int B, N, C;
    int post, pre;                            // 0 none, 1 LayerNorm, 2 RMSNorm
    int gmode, gdt;                           // gate: 0 none, 1 per sample, 2 per token; its dtype
    float eps1, eps2;
    int chunk;                                // rows of one sample per workgroup
    int wanted;                               // backward: bit i: slot i of part is folded afterwards
};

typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x8 all8(float v) { return (f32x8){v, v, v, v, v, v, v, v}; }

// the 8 channels of thread t of a row: 8 t .. 8 t + 7 where rows are 16-byte aligned (VEC), else j TPR + t (neighbouring threads, neighbouring channels);
// channels past C are 0
template <typename T, bool VEC>
__device__ __forceinline__ f32x8 ldv(const T* p, int t, int tpr, int C) {
    f32x8 v = all8(0.f);
    if constexpr (VEC) {
        if (8 * t < C) {
            if constexpr (sizeof(T) == 2) {
                const uint4 u = *reinterpret_cast<const uint4*>(p + 8 * t);
                v = (f32x8){__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u),
                            __uint_as_float(u.z << 16), __uint_as_float(u.z & 0xffff0000u), __uint_as_float(u.w << 16), __uint_as_float(u.w & 0xffff0000u)};
            } else {
                const f32x4 a = load4(p + 8 * t), b = load4(p + 8 * t + 4);
                v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (j * tpr + t < C) v[j] = to_f32(p[j * tpr + t]);
    }
    return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void stv(T* p, int t, int tpr, int C, f32x8 v) {
    if constexpr (VEC) {
        if (8 * t < C) {
            store4(p + 8 * t, __builtin_shufflevector(v, v, 0, 1, 2, 3));
            store4(p + 8 * t + 4, __builtin_shufflevector(v, v, 4, 5, 6, 7));
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (j * tpr + t < C) p[j * tpr + t] = from_f32<T>(v[j]);
    }
}
template <> __device__ __forceinline__ void stv<bf16_t, true>(bf16_t* p, int t, int, int C, f32x8 v) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    if (8 * t < C) *reinterpret_cast<b8*>(p + 8 * t) = __builtin_convertvector(v, b8);
}
// A row as it arrives, converted where it is used: the next step's rows are requested before this step's arithmetic and its barriers
template <typename T, bool VEC> struct Raw {
    static constexpr int N = VEC ? (int)sizeof(T) * 2 : 8;
    unsigned a[N];
    __device__ __forceinline__ void load(const T* row, int t, int tpr, int C) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (row && 8 * t < C) u = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row + 8 * t) + 16 * i);
                a[4 * i] = u.x; a[4 * i + 1] = u.y; a[4 * i + 2] = u.z; a[4 * i + 3] = u.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] = 0u;
                if (row && j * tpr + t < C) {
                    if constexpr (sizeof(T) == 2) a[j] = reinterpret_cast<const uint16_t*>(row)[j * tpr + t];
                    else a[j] = reinterpret_cast<const unsigned*>(row)[j * tpr + t];
                }
            }
        }
    }
    __device__ __forceinline__ f32x8 get() const {
        f32x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(a[j]);
            else if constexpr (!VEC) v[j] = __uint_as_float(a[j] << 16);
            else v[j] = __uint_as_float(j & 1 ? a[j / 2] & 0xffff0000u : a[j / 2] << 16);
        }
        return v;
    }
};
// a gate row: its dtype is a run-time flag (uniform over the launch)
template <bool VEC>
__device__ __forceinline__ f32x8 ldg(const void* p, int dt, long row, int t, int tpr, int C) {
    if (dt == PASSION_BF16) return ldv<bf16_t, VEC>(static_cast<const bf16_t*>(p) + row * C, t, tpr, C);
    return ldv<float, VEC>(static_cast<const float*>(p) + row * C, t, tpr, C);
}
template <bool VEC>
__device__ __forceinline__ f32x8 ldc(const float* p, float other, int t, int tpr, int C) { return p ? ldv<float, VEC>(p, t, tpr, C) : all8(other); }

__device__ __forceinline__ float sum8(f32x8 v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }

struct RowThread { int t, sub, rpb, wv, w0, nw, tpr, lanes; float nwave, invC, invW; f32x8 in; };
template <bool VEC>
__device__ __forceinline__ RowThread row_thread(int tpr, int C) {
    RowThread a;
    a.tpr = tpr;
    a.t = threadIdx.x & (tpr - 1);
    a.sub = threadIdx.x / tpr;
    a.rpb = blockDim.x / tpr;
    a.wv = threadIdx.x >> 6;
    a.nw = tpr > 64 ? tpr >> 6 : 1;
    a.w0 = a.wv / a.nw * a.nw;
    a.lanes = tpr < 64 ? tpr : 64;
#pragma unroll
    for (int j = 0; j < VPT; ++j) a.in[j] = (VEC ? 8 * a.t + j : j * tpr + a.t) < C ? 1.f : 0.f;      // the thread's channels inside C
    a.nwave = lanes_sum(sum8(a.in), 64);                 // those of the whole wavefront (used where a row spans wavefronts)
    a.invC = 1.f / (float)C;
    a.invW = a.nwave > 0.f ? 1.f / a.nwave : 0.f;
    return a;
}

// two sums over the threads of each of NR rows; red: 2 NR floats a wavefront, in use until the second barrier after this one
template <int NR>
__device__ __forceinline__ void row_sum2(float (&x)[NR], float (&y)[NR], const RowThread& a, float* red) {
#pragma unroll
    for (int u = 0; u < NR; ++u) { x[u] = lanes_sum(x[u], a.lanes); y[u] = lanes_sum(y[u], a.lanes); }
    if (a.tpr <= 64) return;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int u = 0; u < NR; ++u) { red[(a.wv * NR + u) * 2] = x[u]; red[(a.wv * NR + u) * 2 + 1] = y[u]; }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        x[u] = y[u] = 0.f;
        for (int i = 0; i < a.nw; ++i) { x[u] += red[((a.w0 + i) * NR + u) * 2]; y[u] += red[((a.w0 + i) * NR + u) * 2 + 1]; }
    }
}

// mean and 1 / sqrt(variance + eps) (kind 1) or 0 and 1 / sqrt(mean square + eps) (kind 2) of NR rows
template <int NR>
__device__ __forceinline__ void moments(const f32x8 (&v)[NR], int kind, float eps, const RowThread& a, float* red, float (&mean)[NR], float (&rstd)[NR]) {
    float s[NR], q[NR];
    if (kind == 2) {
#pragma unroll
        for (int u = 0; u < NR; ++u) { s[u] = 0.f; q[u] = sum8(v[u] * v[u]); }
        row_sum2<NR>(s, q, a, red);
#pragma unroll
        for (int u = 0; u < NR; ++u) { mean[u] = 0.f; rstd[u] = 1.f / sqrtf(q[u] * a.invC + eps); }
        return;
    }
    const float inv = a.tpr <= 64 ? a.invC : a.invW;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        s[u] = lanes_sum(sum8(v[u]), a.lanes);               // channels past C hold 0
        const f32x8 d = (v[u] - s[u] * inv) * a.in;
        q[u] = lanes_sum(sum8(d * d), a.lanes);
    }
    if (a.tpr > 64) {                                        // wavefronts of a row: second moments about their own means, joined about the row's
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                float* r = red + (a.wv * NR + u) * 3;
                r[0] = s[u]; r[1] = q[u]; r[2] = a.nwave;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            s[u] = q[u] = 0.f;
            for (int i = 0; i < a.nw; ++i) s[u] += red[((a.w0 + i) * NR + u) * 3];
            mean[u] = s[u] * a.invC;
            for (int i = 0; i < a.nw; ++i) {
                const float* r = red + ((a.w0 + i) * NR + u) * 3;
                const float n = r[2], d = n > 0.f ? r[0] / n - mean[u] : 0.f;
                q[u] += __builtin_fmaf(n * d, d, r[1]);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < NR; ++u) mean[u] = s[u] * a.invC;
    }
#pragma unroll
    for (int u = 0; u < NR; ++u) rstd[u] = 1.f / sqrtf(q[u] * a.invC + eps);
}

// grid (row chunks, B); a step takes NR rows a row-thread group: their loads are in flight together and they share the barriers
template <typename TX, typename TH, bool VEC, int NT, int NR>
__global__ __launch_bounds__(NT) void rn_fwd_kernel(RnP p, int tpr) {
    __shared__ float red[2][2][NT / 64 * NR * 3];            // [step parity][norm]: a slot is written again two barriers later at the earliest
    const int C = p.C, b = blockIdx.y;
    const RowThread a = row_thread<VEC>(tpr, C);
    const f32x8 w1 = ldc<VEC>(p.w1, 1.f, a.t, tpr, C), b1 = ldc<VEC>(p.b1, 0.f, a.t, tpr, C), w2 = ldc<VEC>(p.w2, 1.f, a.t, tpr, C),
                b2 = ldc<VEC>(p.b2, 0.f, a.t, tpr, C);
    f32x8 sc = ldc<VEC>(p.scale, 1.f, a.t, tpr, C);
    if (p.gmode == 1) sc *= ldg<VEC>(p.gate, p.gdt, b, a.t, tpr, C);
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, p.N);
    int par = 0;
    Raw<TX, VEC> xn[NR];
    Raw<TH, VEC> hn[NR];
    auto fetch = [&](int n0) {
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const long at = ((long)b * p.N + min(n0 + u * a.rpb + a.sub, hi - 1)) * C;
            hn[u].load(static_cast<const TH*>(p.h) + at, a.t, tpr, C);
            xn[u].load(static_cast<const TX*>(p.x) + at, a.t, tpr, C);
        }
    };
    if (lo < hi) fetch(lo);
    for (int n0 = lo; n0 < hi; n0 += a.rpb * NR, par ^= 1) {             // every thread of the workgroup makes the same number of rounds (barriers inside)
        bool ok[NR];
        long row[NR];
        f32x8 xv[NR], hv[NR], gv[NR];
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const int n = n0 + u * a.rpb + a.sub;
            ok[u] = n < hi;
            row[u] = (long)b * p.N + (ok[u] ? n : hi - 1);
            hv[u] = hn[u].get();
            xv[u] = xn[u].get();
            if (p.gmode == 2) gv[u] = ldg<VEC>(p.gate, p.gdt, row[u], a.t, tpr, C);
        }
        if (n0 + a.rpb * NR < hi) fetch(n0 + a.rpb * NR);
        float m1[NR], r1[NR], m2[NR], r2[NR];
#pragma unroll
        for (int u = 0; u < NR; ++u) { m1[u] = m2[u] = 0.f; r1[u] = r2[u] = 1.f; }
        if (p.post) {
            moments<NR>(hv, p.post, p.eps1, a, red[par][0], m1, r1);
#pragma unroll
            for (int u = 0; u < NR; ++u) hv[u] = (hv[u] - m1[u]) * r1[u] * w1 + b1;
        }
#pragma unroll
        for (int u = 0; u < NR; ++u) xv[u] = ((p.gmode == 2 ? hv[u] * gv[u] : hv[u]) * sc + xv[u]) * a.in;
        if (p.pre) {
            moments<NR>(xv, p.pre, p.eps2, a, red[par][1], m2, r2);
#pragma unroll
            for (int u = 0; u < NR; ++u) hv[u] = (xv[u] - m2[u]) * r2[u] * w2 + b2;
        }
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            if (!ok[u]) continue;
            stv<TX, VEC>(static_cast<TX*>(p.r) + row[u] * C, a.t, tpr, C, xv[u]);
            if (p.pre) stv<TH, VEC>(static_cast<TH*>(p.y) + row[u] * C, a.t, tpr, C, hv[u]);
            if (a.t == 0 && p.stat) store4(p.stat + 4 * row[u], (f32x4){m1[u], r1[u], m2[u], r2[u]});
        }
    }
}

template <typename TX, typename TH, bool VEC, int NT, int NR>
__global__ __launch_bounds__(NT) void rn_bwd_kernel(RnP p, int tpr) {
    __shared__ float red[2][2][NT / 64 * NR * 2];
    extern __shared__ __attribute__((aligned(16))) float fold[];                     // [rpb][tpr][8], only where a workgroup holds several rows
    const int C = p.C, b = blockIdx.y;
    const RowThread a = row_thread<VEC>(tpr, C);
    const f32x8 w1 = ldc<VEC>(p.w1, 1.f, a.t, tpr, C), b1 = ldc<VEC>(p.b1, 0.f, a.t, tpr, C), w2 = ldc<VEC>(p.w2, 1.f, a.t, tpr, C),
                sc = ldc<VEC>(p.scale, 1.f, a.t, tpr, C);
    f32x8 g[NR], acc[6];
#pragma unroll
    for (int u = 0; u < NR; ++u) g[u] = p.gmode == 1 ? ldg<VEC>(p.gate, p.gdt, b, a.t, tpr, C) : all8(1.f);
#pragma unroll
    for (int i = 0; i < 6; ++i) acc[i] = all8(0.f);
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, p.N);
    int par = 0;
    Raw<TX, VEC> xn[NR], drn[NR];
    Raw<TH, VEC> hn[NR], dyn[NR];
    f32x4 stn[NR];
    auto fetch = [&](int n0) {
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const int n = n0 + u * a.rpb + a.sub;
            const bool in = n < hi;
            const long r = (long)b * p.N + (in ? n : hi - 1), at = r * C;
            stn[u] = load4(p.stat + 4 * r);
            hn[u].load(static_cast<const TH*>(p.h) + at, a.t, tpr, C);
            xn[u].load(static_cast<const TX*>(p.x) + at, a.t, tpr, C);
            drn[u].load(in && p.dr ? static_cast<const TX*>(p.dr) + at : nullptr, a.t, tpr, C);
            dyn[u].load(in && p.dy ? static_cast<const TH*>(p.dy) + at : nullptr, a.t, tpr, C);
        }
    };
    if (lo < hi) fetch(lo);
    for (int n0 = lo; n0 < hi; n0 += a.rpb * NR, par ^= 1) {
        bool ok[NR];
        long row[NR];
        f32x8 xv[NR], hv[NR], dr[NR], dy[NR], uu[NR];
        f32x4 st[NR];
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const int n = n0 + u * a.rpb + a.sub;
            ok[u] = n < hi;
            row[u] = (long)b * p.N + (ok[u] ? n : hi - 1);
            st[u] = stn[u];
            hv[u] = hn[u].get();
            xv[u] = xn[u].get();
            dr[u] = drn[u].get();
            dy[u] = dyn[u].get();
            if (p.gmode == 2) g[u] = ldg<VEC>(p.gate, p.gdt, row[u], a.t, tpr, C);
        }
        if (n0 + a.rpb * NR < hi) fetch(n0 + a.rpb * NR);
        float s1[NR], s2[NR];
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            hv[u] = (hv[u] - st[u][0]) * st[u][1];                          // h hat (h itself without a post norm: mean 0, rstd 1)
            uu[u] = hv[u] * w1 + b1;
            if (p.pre) xv[u] = (uu[u] * g[u] * sc + xv[u] - st[u][2]) * st[u][3];       // r hat
        }
        if (p.pre && p.dy) {                                                // dr += d pre(r) / d r
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                acc[2] += dy[u] * xv[u];
                acc[3] += dy[u];
                dy[u] = dy[u] * w2 * a.in;
                s1[u] = sum8(dy[u] * xv[u]);
                s2[u] = sum8(dy[u]);
            }
            row_sum2<NR>(s1, s2, a, red[par][0]);
#pragma unroll
            for (int u = 0; u < NR; ++u) dr[u] += (dy[u] - (p.pre == 1 ? s2[u] * a.invC : 0.f) - xv[u] * (s1[u] * a.invC)) * st[u][3];
        }
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            if (ok[u]) stv<TX, VEC>(static_cast<TX*>(p.dx) + row[u] * C, a.t, tpr, C, dr[u]);
            else dr[u] = all8(0.f);
            acc[4] += dr[u] * (uu[u] * g[u]);
            const f32x8 dm = dr[u] * sc;
            uu[u] *= dm;                                                    // gradient of the gate
            acc[5] += uu[u];
            dy[u] = dm * g[u];                                              // ... of post(h)
            acc[0] += dy[u] * hv[u];
            acc[1] += dy[u];
            dy[u] = dy[u] * w1;
            if (ok[u] && p.dgate_tok) {
                if (p.gdt == PASSION_BF16) stv<bf16_t, VEC>(static_cast<bf16_t*>(p.dgate_tok) + row[u] * C, a.t, tpr, C, uu[u]);
                else stv<float, VEC>(static_cast<float*>(p.dgate_tok) + row[u] * C, a.t, tpr, C, uu[u]);
            }
        }
        if (p.post) {
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                const f32x8 d = dy[u] * a.in;
                s1[u] = sum8(d * hv[u]);
                s2[u] = sum8(d);
            }
            row_sum2<NR>(s1, s2, a, red[par][1]);
#pragma unroll
            for (int u = 0; u < NR; ++u) dy[u] = (dy[u] - (p.post == 1 ? s2[u] * a.invC : 0.f) - hv[u] * (s1[u] * a.invC)) * st[u][1];
        }
#pragma unroll
        for (int u = 0; u < NR; ++u)
            if (ok[u]) stv<TH, VEC>(static_cast<TH*>(p.dh) + row[u] * C, a.t, tpr, C, dy[u]);
    }
    float* out = p.part + ((long)b * gridDim.x + blockIdx.x) * 6 * C;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        if (!((p.wanted >> i) & 1)) continue;                         // uniform
        if (a.rpb > 1) {                                              // rows of the workgroup, in order
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; ++j) fold[(j * a.rpb + a.sub) * tpr + a.t] = acc[i][j];
            __syncthreads();
            for (int e = threadIdx.x; e < VPT * tpr; e += NT) {
                const int j = e / tpr, t = e % tpr, c = VEC ? 8 * t + j : j * tpr + t;
                float s = 0.f;
                for (int r = 0; r < a.rpb; ++r) s += fold[(j * a.rpb + r) * tpr + t];
                if (c < C) out[(long)i * C + c] = s;
            }
        } else stv<float, VEC>(out + (long)i * C, a.t, tpr, C, acc[i]);
    }
}

// column sums of the partials: slot 0 .. 4 over all workgroups, the gate's (slot 5) over those of its sample.  32 columns x 32 runs of
// partials a workgroup, joined in order.  grid (ceil(C / 32), 5 + B)
struct RnFold { const float* part; float* out[5]; void* dgate; int gdt, C, nblk, B; };
__global__ __launch_bounds__(1024) void rn_fold_kernel(RnFold f) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, run = threadIdx.x >> 5;
    const int what = blockIdx.y < 5 ? blockIdx.y : 5, b = blockIdx.y - 5;
    if (what < 5 ? !f.out[what] : !f.dgate) return;                   // uniform over the workgroup
    const long lo = what < 5 ? 0 : (long)b * f.nblk, n = what < 5 ? (long)f.B * f.nblk : f.nblk;
    const long i0 = lo + n * run / 32, i1 = lo + n * (run + 1) / 32;
    float s = 0.f;
    if (c < f.C) {
        long i = i0;
        for (; i + 4 <= i1; i += 4) {                                 // four loads in flight, added in order
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = f.part[((i + u) * 6 + what) * f.C + c];
#pragma unroll
            for (int u = 0; u < 4; ++u) s += v[u];
        }
        for (; i < i1; ++i) s += f.part[(i * 6 + what) * f.C + c];
    }
    red[run][lane] = s;
    __syncthreads();
    if (run == 0 && c < f.C) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][lane];
        if (what < 5) f.out[what][c] = s;
        else if (f.gdt == PASSION_BF16) static_cast<bf16_t*>(f.dgate)[(long)b * f.C + c] = (bf16_t)s;
        else static_cast<float*>(f.dgate)[(long)b * f.C + c] = s;
    }
}

int threads_per_row(int C) {
    int t = 1;
    while (t * VPT < C) t *= 2;
    return t;
}

// rows of one sample a workgroup, whole rounds of its rows: at most 2048 workgroups forward (8 x 4096 x 2048 bf16 145 us, by 1024 157, by 4096 137; 12003 x 768 f32 49, 40, 42; 20000 x 256 bf16
// 13.3, 17.2, 19.9) and 1024 backward, each of which leaves a row of column sums (forward + backward there 319 us, by 512 307, by 2048 326; 104, 97, 117; 39.6, 34.8, 42.5)
int pick_chunk(int B, int N, int rpb, int target) {
    const long want = (long)target / B > 0 ? target / B : 1;
    long chunk = (N + want - 1) / want;
    chunk = (chunk + rpb - 1) / rpb * rpb;
    return (int)(chunk < 1 ? rpb : chunk);
}

template <typename TX, typename TH, int NT>
int launch_nt(const RnP& p, int tpr, bool bwd, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)(((long)p.N + p.chunk - 1) / p.chunk), p.B);
    if (bwd) {
        const int bytes = NT > tpr ? NT * VPT * (int)sizeof(float) : 0;
        if (vec) hipLaunchKernelGGL((rn_bwd_kernel<TX, TH, true, NT, 1>), grid, dim3(NT), bytes, st, p, tpr);
        else hipLaunchKernelGGL((rn_bwd_kernel<TX, TH, false, NT, 1>), grid, dim3(NT), bytes, st, p, tpr);
    } else {
        if (vec) hipLaunchKernelGGL((rn_fwd_kernel<TX, TH, true, NT, NT == 1024 ? 1 : 2>), grid, dim3(NT), 0, st, p, tpr);
        else hipLaunchKernelGGL((rn_fwd_kernel<TX, TH, false, NT, 1>), grid, dim3(NT), 0, st, p, tpr);
    }
    LAUNCH_RET();
    return 0;
}
template <typename TX, typename TH>
int launch(const RnP& p, bool bwd, bool vec, hipStream_t st) {
    const int tpr = threads_per_row(p.C);
    if (tpr <= 256) return launch_nt<TX, TH, 256>(p, tpr, bwd, vec, st);
    return tpr == 512 ? launch_nt<TX, TH, 512>(p, tpr, bwd, vec, st) : launch_nt<TX, TH, 1024>(p, tpr, bwd, vec, st);
}

int dispatch(const RnP& p, int xdt, int hdt, bool bwd, hipStream_t st) {
    uintptr_t bits = (uintptr_t)p.x | (uintptr_t)p.h | (uintptr_t)p.gate | (uintptr_t)p.w1 | (uintptr_t)p.b1 | (uintptr_t)p.w2 | (uintptr_t)p.b2 | (uintptr_t)p.scale |
                     (uintptr_t)p.r | (uintptr_t)p.y | (uintptr_t)p.dr | (uintptr_t)p.dy | (uintptr_t)p.dx | (uintptr_t)p.dh | (uintptr_t)p.dgate_tok | (uintptr_t)p.part;
    const bool vec = p.C % 8 == 0 && !(bits & 15);
    if (xdt == PASSION_F32 && hdt == PASSION_F32) return launch<float, float>(p, bwd, vec, st);
    if (xdt == PASSION_F32 && hdt == PASSION_BF16) return launch<float, bf16_t>(p, bwd, vec, st);
    if (xdt == PASSION_BF16 && hdt == PASSION_BF16) return launch<bf16_t, bf16_t>(p, bwd, vec, st);
    return -1003;
}

bool bad_args(int B, int N, int C, int post, int pre, int gmode, int gdt) {
    return B < 1 || B > 65530 || N < 1 || N > RN_MAX_N || C < 1 || C > RN_MAX_C || post < 0 || post > 2 || pre < 0 || pre > 2 || gmode < 0 || gmode > 2 ||
           (gdt != PASSION_F32 && gdt != PASSION_BF16);
}

constexpr int BWD_TARGET = 1024;
int bwd_blocks(int B, int N, int C, int& chunk) {
    const int tpr = threads_per_row(C), rpb = (tpr < 256 ? 256 : tpr) / tpr;
    chunk = pick_chunk(B, N, rpb, BWD_TARGET);
    return (int)(((long)N + chunk - 1) / chunk);
}

}  // namespace

extern "C" int64_t passion_residual_norm_part_floats(int B, int N, int C) {
    if (bad_args(B, N, C, 0, 0, 0, 0)) return -1003;
    int chunk;
    return (int64_t)B * bwd_blocks(B, N, C, chunk) * 6 * C;
}

extern "C" int passion_residual_norm_fwd(const void* x, int x_dtype, const void* h, int h_dtype, const float* w_post, const float* b_post, int post,
                                         float eps_post, const void* gate, int gate_mode, int gate_dtype, const float* scale, const float* w_pre,
                                         const float* b_pre, int pre, float eps_pre, int B, int N, int C, void* r, void* y, float* stat, void* stream) {
    if (bad_args(B, N, C, post, pre, gate_mode, gate_dtype) || !x || !h || !r || (pre && !y) || (gate_mode && !gate)) return -1003;
    RnP p{};
    p.x = x; p.h = h; p.gate = gate; p.w1 = post ? w_post : nullptr; p.b1 = post == 1 ? b_post : nullptr; p.w2 = w_pre; p.b2 = pre == 1 ? b_pre : nullptr;
    p.scale = scale; p.r = r; p.y = y; p.stat = stat; p.B = B; p.N = N; p.C = C; p.post = post; p.pre = pre; p.gmode = gate_mode; p.gdt = gate_dtype;
    p.eps1 = eps_post; p.eps2 = eps_pre;
    const int tpr = threads_per_row(C), rpb = (tpr < 256 ? 256 : tpr) / tpr;
    p.chunk = pick_chunk(B, N, rpb, 2048);
    return dispatch(p, x_dtype, h_dtype, false, (hipStream_t)stream);
}

extern "C" int passion_residual_norm_bwd(const void* x, int x_dtype, const void* h, int h_dtype, const float* w_post, const float* b_post, int post,
                                         const void* gate, int gate_mode, int gate_dtype, const float* scale, const float* w_pre, int pre,
                                         const float* stat, const void* dr, const void* dy, int B, int N, int C, void* dx, void* dh, void* dgate,
                                         float* dw_post, float* db_post, float* dw_pre, float* db_pre, float* dscale, float* part, void* stream) {
    if (bad_args(B, N, C, post, pre, gate_mode, gate_dtype) || !x || !h || !stat || !dx || !dh || !part || (gate_mode && !gate)) return -1003;
    RnP p{};
    p.x = x; p.h = h; p.gate = gate; p.w1 = post ? w_post : nullptr; p.b1 = post == 1 ? b_post : nullptr; p.w2 = w_pre; p.scale = scale;
    p.stat = const_cast<float*>(stat); p.dr = dr; p.dy = pre ? dy : nullptr; p.dx = dx; p.dh = dh; p.dgate_tok = gate_mode == 2 ? dgate : nullptr;
    p.part = part; p.B = B; p.N = N; p.C = C; p.post = post; p.pre = pre; p.gmode = gate_mode; p.gdt = gate_dtype;
    p.wanted = (dw_post ? 1 : 0) | (db_post ? 2 : 0) | (dw_pre ? 4 : 0) | (db_pre ? 8 : 0) | (dscale ? 16 : 0) | (gate_mode == 1 && dgate ? 32 : 0);
    const int nblk = bwd_blocks(B, N, C, p.chunk);
    hipStream_t st = (hipStream_t)stream;
    const int rc = dispatch(p, x_dtype, h_dtype, true, st);
    if (rc) return rc;
    RnFold f{part, {dw_post, db_post, dw_pre, db_pre, dscale}, gate_mode == 1 ? dgate : nullptr, gate_dtype, C, nblk, B};
    if (p.wanted) {
        hipLaunchKernelGGL(rn_fold_kernel, dim3((C + 31) / 32, 5 + (gate_mode == 1 && dgate ? B : 0)), dim3(1024), 0, st, f);
        LAUNCH_RET();
    }
    return 0;
}
