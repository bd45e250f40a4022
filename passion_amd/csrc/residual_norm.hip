// The residual step between two transformer blocks, one launch each way:
//     u = post(h),   r = x + scale * gate * u,   y = pre(r)
// h: a block's output, x: the residual stream, post / pre: LayerNorm or RMSNorm over the C channels (each optional), gate: per sample
// and channel or per token and channel, scale: per channel.  The glue of the reference's Transformer (code/models/mmformer.py:230-256,
// 284-300: x + dropout(f(norm(x))), norm of the next block) in the form a gated, post-normed block has it.
//
// Bound by HBM: forward reads x, h (, a token gate) and writes r, y once; backward reads x, h, dr, dy and writes dx, dh.  The backward
// forms r again from x and h instead of reading it: the same bytes, and the parameter gradients see the unrounded r.
//
// Layout: a row = C channels over TPR threads (a power of two, 8 channels a thread: one 16-byte access a thread and bf16 tensor), 256 / TPR
// rows a workgroup (one row from TPR = 256 on).  Rows of up to 512 channels live inside one wavefront: moments by butterfly shuffles.
// Wider ones exchange (sum, second moment about the wavefront's own mean) through LDS and join them in wavefront order -- one barrier
// a norm and no cancellation in the variance.  Channel vectors (weights, scale, a sample's gate) stay in registers over a workgroup's rows.
// Column sums of the backward: in registers over the workgroup's rows (of one sample), one partial per workgroup, folded in
// workgroup order by a second kernel: no atomics, results repeat bit for bit.
// All arithmetic and every sum is f32; x, h, y, r and the gradients round once when they are stored.
#include "common.h"
#include "passion_hip.h"

namespace {

constexpr int RN_MAX_C = 8192, VPT = 8;

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
};

// channel j of thread t of a row: 8 t + j where rows are 16-byte aligned (VEC), else j TPR + t (neighbouring threads, neighbouring channels)
template <bool VEC> __device__ __forceinline__ int chan(int t, int j, int tpr) { return VEC ? 8 * t + j : j * tpr + t; }

template <typename T, bool VEC>
__device__ __forceinline__ void ldv(const T* p, int t, int tpr, int C, float (&v)[VPT]) {
    if constexpr (VEC) {
        if (8 * t < C) {
            if constexpr (sizeof(T) == 2) VecIO<bf16_t, 8>::load(reinterpret_cast<const bf16_t*>(p) + 8 * t, v);
            else {
                const f32x4 a = load4(reinterpret_cast<const float*>(p) + 8 * t), b = load4(reinterpret_cast<const float*>(p) + 8 * t + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) { const int c = chan<false>(t, j, tpr); v[j] = c < C ? to_f32(p[c]) : 0.f; }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void stv(T* p, int t, int tpr, int C, const float (&v)[VPT]) {
    if constexpr (VEC) {
        if (8 * t < C) {
            if constexpr (sizeof(T) == 2) VecIO<bf16_t, 8>::store(reinterpret_cast<bf16_t*>(p) + 8 * t, v);
            else {
                store4(reinterpret_cast<float*>(p) + 8 * t, (f32x4){v[0], v[1], v[2], v[3]});
                store4(reinterpret_cast<float*>(p) + 8 * t + 4, (f32x4){v[4], v[5], v[6], v[7]});
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) { const int c = chan<false>(t, j, tpr); if (c < C) p[c] = from_f32<T>(v[j]); }
    }
}
// a gate row: its dtype is a run-time flag (uniform over the launch)
template <bool VEC>
__device__ __forceinline__ void ldg(const void* p, int dt, long row, int t, int tpr, int C, float (&v)[VPT]) {
    if (dt == PASSION_BF16) ldv<bf16_t, VEC>(static_cast<const bf16_t*>(p) + row * C, t, tpr, C, v);
    else ldv<float, VEC>(static_cast<const float*>(p) + row * C, t, tpr, C, v);
}
template <bool VEC>
__device__ __forceinline__ void ldc(const float* p, float other, int t, int tpr, int C, float (&v)[VPT]) {
    if (p) ldv<float, VEC>(p, t, tpr, C, v);
    else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) v[j] = other;
    }
}

// two sums over the threads of a row.  red: [rows of the workgroup][2 wavefront slots ...], one use per barrier interval
__device__ __forceinline__ void row_sum2(float& a, float& b, int tpr, float* red, int wv) {
    const int w = tpr < 64 ? tpr : 64;
    for (int o = w >> 1; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
    if (tpr <= 64) return;
    const int nw = tpr >> 6, w0 = wv / nw * nw;
    if ((threadIdx.x & 63) == 0) { red[2 * wv] = a; red[2 * wv + 1] = b; }
    __syncthreads();
    a = b = 0.f;
    for (int i = 0; i < nw; ++i) { a += red[2 * (w0 + i)]; b += red[2 * (w0 + i) + 1]; }
}

// mean and 1 / sqrt(variance + eps) (LayerNorm) or 0 and 1 / sqrt(mean square + eps) of a row; nval: the thread's channels inside C,
// nwave: those of the whole wavefront's part of the row
__device__ __forceinline__ void moments(const float (&v)[VPT], int nval, float nwave, int kind, float eps, float invC, int tpr, float* red, int wv,
                                        float& mean, float& rstd) {
    float s = 0.f, q = 0.f;
    if (kind == 2) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) q = __builtin_fmaf(v[j], v[j], q);
        row_sum2(s, q, tpr, red, wv);
        mean = 0.f;
        rstd = 1.f / sqrtf(q * invC + eps);
        return;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) s += v[j];                      // channels past C hold 0
    const int w = tpr < 64 ? tpr : 64;
    for (int o = w >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    const float mw = tpr <= 64 ? s * invC : (nwave > 0.f ? s / nwave : 0.f);
#pragma unroll
    for (int j = 0; j < VPT; ++j) { const float d = v[j] - mw; if (j < nval) q = __builtin_fmaf(d, d, q); }
    for (int o = w >> 1; o > 0; o >>= 1) q += __shfl_xor(q, o, 64);
    if (tpr > 64) {
        const int nw = tpr >> 6, w0 = wv / nw * nw;
        if ((threadIdx.x & 63) == 0) { red[3 * wv] = s; red[3 * wv + 1] = q; red[3 * wv + 2] = nwave; }
        __syncthreads();
        s = 0.f;
        for (int i = 0; i < nw; ++i) s += red[3 * (w0 + i)];
        mean = s * invC;
        q = 0.f;
        for (int i = 0; i < nw; ++i) {
            const float n = red[3 * (w0 + i) + 2], d = n > 0.f ? red[3 * (w0 + i)] / n - mean : 0.f;
            q += __builtin_fmaf(n * d, d, red[3 * (w0 + i) + 1]);
        }
    } else mean = mw;
    rstd = 1.f / sqrtf(q * invC + eps);
}

struct RowThread { int t, sub, rpb, nval; float nwave; };
template <bool VEC>
__device__ __forceinline__ RowThread row_thread(int tpr, int C) {
    RowThread a;
    a.t = threadIdx.x & (tpr - 1);
    a.sub = threadIdx.x / tpr;
    a.rpb = blockDim.x / tpr;
    if (VEC) a.nval = 8 * a.t < C ? 8 : 0;
    else a.nval = C > a.t ? min(VPT, (C - a.t + tpr - 1) / tpr) : 0;
    float n = (float)a.nval;
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    a.nwave = n;                                      // used where a row spans wavefronts only
    return a;
}

// grid (row chunks, B)
template <typename TX, typename TH, bool VEC, int NT>
__global__ __launch_bounds__(NT) void rn_fwd_kernel(RnP p, int tpr) {
    __shared__ float red[2][16 * 3];
    const int wv = threadIdx.x >> 6, C = p.C, b = blockIdx.y;
    const RowThread a = row_thread<VEC>(tpr, C);
    const float invC = 1.f / (float)C;
    float w1[VPT], b1[VPT], w2[VPT], b2[VPT], sc[VPT], g[VPT];
    ldc<VEC>(p.w1, 1.f, a.t, tpr, C, w1);
    ldc<VEC>(p.b1, 0.f, a.t, tpr, C, b1);
    ldc<VEC>(p.w2, 1.f, a.t, tpr, C, w2);
    ldc<VEC>(p.b2, 0.f, a.t, tpr, C, b2);
    ldc<VEC>(p.scale, 1.f, a.t, tpr, C, sc);
    if (p.gmode == 1) {
        ldg<VEC>(p.gate, p.gdt, b, a.t, tpr, C, g);
#pragma unroll
        for (int j = 0; j < VPT; ++j) sc[j] *= g[j];
    }
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, p.N);
    for (int n0 = lo; n0 < hi; n0 += a.rpb) {                    // every thread of the workgroup makes the same number of rounds (barriers inside)
        const bool ok = n0 + a.sub < hi;
        const long row = (long)b * p.N + (ok ? n0 + a.sub : hi - 1);
        float xv[VPT], hv[VPT];
        ldv<TX, VEC>(static_cast<const TX*>(p.x) + row * C, a.t, tpr, C, xv);
        ldv<TH, VEC>(static_cast<const TH*>(p.h) + row * C, a.t, tpr, C, hv);
        if (p.gmode == 2) ldg<VEC>(p.gate, p.gdt, row, a.t, tpr, C, g);
        float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
        if (p.post) {
            moments(hv, a.nval, a.nwave, p.post, p.eps1, invC, tpr, red[0], wv, m1, r1);
#pragma unroll
            for (int j = 0; j < VPT; ++j) hv[j] = __builtin_fmaf((hv[j] - m1) * r1, w1[j], b1[j]);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const float m = p.gmode == 2 ? hv[j] * g[j] : hv[j];
            xv[j] = j < a.nval ? __builtin_fmaf(m, sc[j], xv[j]) : 0.f;
        }
        if (p.pre) {
            moments(xv, a.nval, a.nwave, p.pre, p.eps2, invC, tpr, red[1], wv, m2, r2);
#pragma unroll
            for (int j = 0; j < VPT; ++j) hv[j] = __builtin_fmaf((xv[j] - m2) * r2, w2[j], b2[j]);
        }
        if (ok) {
            stv<TX, VEC>(static_cast<TX*>(p.r) + row * C, a.t, tpr, C, xv);
            if (p.pre) stv<TH, VEC>(static_cast<TH*>(p.y) + row * C, a.t, tpr, C, hv);
            if (a.t == 0 && p.stat) store4(p.stat + 4 * row, (f32x4){m1, r1, m2, r2});
        }
        if (tpr > 64) __syncthreads();               // the slots are free for the next row
    }
}

template <typename TX, typename TH, bool VEC, int NT>
__global__ __launch_bounds__(NT) void rn_bwd_kernel(RnP p, int tpr) {
    __shared__ float red[2][16 * 2];
    extern __shared__ __attribute__((aligned(16))) float fold[];                     // [rpb][tpr][8], only where a workgroup holds several rows
    const int wv = threadIdx.x >> 6, C = p.C, b = blockIdx.y;
    const RowThread a = row_thread<VEC>(tpr, C);
    const float invC = 1.f / (float)C;
    float w1[VPT], b1[VPT], w2[VPT], sc[VPT], g[VPT];
    ldc<VEC>(p.w1, 1.f, a.t, tpr, C, w1);
    ldc<VEC>(p.b1, 0.f, a.t, tpr, C, b1);
    ldc<VEC>(p.w2, 1.f, a.t, tpr, C, w2);
    ldc<VEC>(p.scale, 1.f, a.t, tpr, C, sc);
    if (p.gmode == 1) ldg<VEC>(p.gate, p.gdt, b, a.t, tpr, C, g);
    else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) g[j] = 1.f;
    }
    float acc[6][VPT];
#pragma unroll
    for (int i = 0; i < 6; ++i)
#pragma unroll
        for (int j = 0; j < VPT; ++j) acc[i][j] = 0.f;
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, p.N);
    for (int n0 = lo; n0 < hi; n0 += a.rpb) {
        const bool ok = n0 + a.sub < hi;
        const long row = (long)b * p.N + (ok ? n0 + a.sub : hi - 1);
        float xv[VPT], hv[VPT], dr[VPT], dy[VPT];
        ldv<TX, VEC>(static_cast<const TX*>(p.x) + row * C, a.t, tpr, C, xv);
        ldv<TH, VEC>(static_cast<const TH*>(p.h) + row * C, a.t, tpr, C, hv);
#pragma unroll
        for (int j = 0; j < VPT; ++j) { dr[j] = 0.f; dy[j] = 0.f; }
        if (ok && p.dr) ldv<TX, VEC>(static_cast<const TX*>(p.dr) + row * C, a.t, tpr, C, dr);
        if (ok && p.dy) ldv<TH, VEC>(static_cast<const TH*>(p.dy) + row * C, a.t, tpr, C, dy);
        if (p.gmode == 2) ldg<VEC>(p.gate, p.gdt, row, a.t, tpr, C, g);
        const f32x4 st = load4(p.stat + 4 * row);
        float u[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            hv[j] = (hv[j] - st[0]) * st[1];                          // h hat (h itself without a post norm: mean 0, rstd 1)
            u[j] = __builtin_fmaf(hv[j], w1[j], b1[j]);
            if (p.pre) {
                const float rr = __builtin_fmaf(u[j] * g[j], sc[j], xv[j]);
                xv[j] = (rr - st[2]) * st[3];                         // r hat
            }
        }
        if (p.pre && p.dy) {                                          // dr += d pre(r) / d r
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                acc[2][j] = __builtin_fmaf(dy[j], xv[j], acc[2][j]);
                acc[3][j] += dy[j];
                dy[j] *= w2[j];
                if (j < a.nval) { s1 = __builtin_fmaf(dy[j], xv[j], s1); s2 += dy[j]; }
            }
            row_sum2(s1, s2, tpr, red[0], wv);
            s1 *= invC;
            s2 = p.pre == 1 ? s2 * invC : 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) dr[j] += st[3] * (dy[j] - s2 - xv[j] * s1);
        }
        if (ok) stv<TX, VEC>(static_cast<TX*>(p.dx) + row * C, a.t, tpr, C, dr);
        else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) dr[j] = 0.f;
        }
        float du[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            acc[4][j] = __builtin_fmaf(dr[j], u[j] * g[j], acc[4][j]);
            const float dm = dr[j] * sc[j];
            u[j] *= dm;                                               // gradient of the gate
            acc[5][j] += u[j];
            du[j] = dm * g[j];
            acc[0][j] = __builtin_fmaf(du[j], hv[j], acc[0][j]);
            acc[1][j] += du[j];
            du[j] *= w1[j];
        }
        if (ok && p.dgate_tok) {
            if (p.gdt == PASSION_BF16) stv<bf16_t, VEC>(static_cast<bf16_t*>(p.dgate_tok) + row * C, a.t, tpr, C, u);
            else stv<float, VEC>(static_cast<float*>(p.dgate_tok) + row * C, a.t, tpr, C, u);
        }
        if (p.post) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (j < a.nval) { s1 = __builtin_fmaf(du[j], hv[j], s1); s2 += du[j]; }
            row_sum2(s1, s2, tpr, red[1], wv);
            s1 *= invC;
            s2 = p.post == 1 ? s2 * invC : 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) du[j] = st[1] * (du[j] - s2 - hv[j] * s1);
        }
        if (ok) stv<TH, VEC>(static_cast<TH*>(p.dh) + row * C, a.t, tpr, C, du);
        if (tpr > 64) __syncthreads();
    }
    float* out = p.part + ((long)b * gridDim.x + blockIdx.x) * 6 * C;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        if (a.rpb > 1) {                                              // rows of the workgroup, in order
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; ++j) fold[(a.sub * tpr + a.t) * VPT + j] = acc[i][j];
            __syncthreads();
            if (a.sub == 0) {
                for (int s = 1; s < a.rpb; ++s)
#pragma unroll
                    for (int j = 0; j < VPT; ++j) acc[i][j] += fold[(s * tpr + a.t) * VPT + j];
            }
        }
        if (a.sub == 0) stv<float, VEC>(out + (long)i * C, a.t, tpr, C, acc[i]);
    }
}

// column sums of the partials: slot 0 .. 4 over all workgroups, the gate's (slot 5) over those of its sample.  64 columns x 4 runs of
// partials a workgroup, joined in order.  grid (ceil(C / 64), 5 + B)
struct RnFold { const float* part; float* out[5]; void* dgate; int gdt, C, nblk, B; };
__global__ __launch_bounds__(256) void rn_fold_kernel(RnFold f) {
    __shared__ float red[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
    const int what = blockIdx.y < 5 ? blockIdx.y : 5, b = blockIdx.y - 5;
    if (what < 5 ? !f.out[what] : !f.dgate) return;                   // uniform over the workgroup
    const long lo = what < 5 ? 0 : (long)b * f.nblk, n = what < 5 ? (long)f.B * f.nblk : f.nblk;
    const long i0 = lo + n * run / 4, i1 = lo + n * (run + 1) / 4;
    float s = 0.f;
    if (c < f.C)
        for (long i = i0; i < i1; ++i) s += f.part[(i * 6 + what) * f.C + c];
    red[run][threadIdx.x & 63] = s;
    __syncthreads();
    if (run == 0 && c < f.C) {
        s = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
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

// rows of one sample a workgroup: enough workgroups for two to four per CU, whole rounds of its rows
int pick_chunk(int B, int N, int rpb, int target) {
    const long want = (long)target / B > 0 ? target / B : 1;
    long chunk = (N + want - 1) / want;
    chunk = (chunk + rpb - 1) / rpb * rpb;
    return (int)(chunk < 1 ? rpb : chunk);
}

template <typename TX, typename TH, int NT>
int launch_nt(const RnP& p, int tpr, bool bwd, bool vec, hipStream_t st) {
    const dim3 grid((p.N + p.chunk - 1) / p.chunk, p.B);
    if (bwd) {
        const int bytes = NT > tpr ? NT * VPT * (int)sizeof(float) : 0;
        if (vec) hipLaunchKernelGGL((rn_bwd_kernel<TX, TH, true, NT>), grid, dim3(NT), bytes, st, p, tpr);
        else hipLaunchKernelGGL((rn_bwd_kernel<TX, TH, false, NT>), grid, dim3(NT), bytes, st, p, tpr);
    } else {
        if (vec) hipLaunchKernelGGL((rn_fwd_kernel<TX, TH, true, NT>), grid, dim3(NT), 0, st, p, tpr);
        else hipLaunchKernelGGL((rn_fwd_kernel<TX, TH, false, NT>), grid, dim3(NT), 0, st, p, tpr);
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
    return B < 1 || B > 65530 || N < 1 || C < 1 || C > RN_MAX_C || post < 0 || post > 2 || pre < 0 || pre > 2 || gmode < 0 || gmode > 2 ||
           (gdt != PASSION_F32 && gdt != PASSION_BF16);
}

constexpr int BWD_TARGET = 1024;
int bwd_blocks(int B, int N, int C, int& chunk) {
    const int tpr = threads_per_row(C), rpb = (tpr < 256 ? 256 : tpr) / tpr;
    chunk = pick_chunk(B, N, rpb, BWD_TARGET);
    return (N + chunk - 1) / chunk;
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
    const int nblk = bwd_blocks(B, N, C, p.chunk);
    hipStream_t st = (hipStream_t)stream;
    const int rc = dispatch(p, x_dtype, h_dtype, true, st);
    if (rc) return rc;
    RnFold f{part, {dw_post, db_post, dw_pre, db_pre, dscale}, gate_mode == 1 ? dgate : nullptr, gate_dtype, C, nblk, B};
    hipLaunchKernelGGL(rn_fold_kernel, dim3((C + 63) / 64, 5 + (gate_mode == 1 && dgate ? B : 0)), dim3(256), 0, st, f);
    LAUNCH_RET();
    return 0;
}
