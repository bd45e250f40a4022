// Distillation from a teacher's top K logits over V classes (the full-distribution form: temp_kl_loss_bs, reference
// code/utils/criterions.py:92-103).  Per row, with p = softmax(teacher / T) over the row's valid entries and q = softmax(student / T) over
// all classes:
//     loss = T^2 sum_k p_k (log p_k - log q_{idx_k}),      d loss / d student = T (q - scatter_add(p))
// An entry whose index is not in [0, V) or whose logit is -inf is absent; a row with no entry left has loss 0 and gradient 0 and its
// student logits are not read by the backward.  The same class may be named twice: both shares count.
//
// Bound by HBM: forward reads the logits once (running maximum and sum in one pass) and keeps one log-sum-exp a row; backward reads them
// once more and writes the gradient once.
//  * V > 512: a workgroup a row, 16-byte accesses between the row's alignment points (a row of an odd width starts anywhere).  The backward
//    stores T g q for the whole row, then the first wavefronts store the K named classes again with p taken off (equal indices merged, one
//    writer each): the bulk of the row needs no comparison with the indices.
//  * V <= 512: G lanes a row (a power of two), the row in registers, 256 / G rows a workgroup -- the voxel classes of this framework (V = 4: one
//    lane, one 16-byte load a row).
// Sums and exponentials are f32; the gradient rounds once.  Exponents are differences of logits times log2(e) / T, and a row's largest logit and the log of its sum stay
// apart: masked classes may hold their type's lowest value (log2(e) / T times that is past the type's range below T = 1.44), and a large common offset costs no bits.
// 4096 x 50000 bf16, K = 32: forward 119 us (3.44 TB/s; a large library maximum or sum, reading alone as well, reaches 3.7 to 4.0), backward 160 (5.1 TB/s of reads and writes).
// The row form against the register form at V <= 512, f32, K = 4, with the gradient: 200000 x 104 689 / 92 us, 100000 x 512 383 / 193, 64 x 512 8.2 / 10.1.
#include "common.h"
#include "passion_hip.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr int SMALL_V = 512, MAX_K = 1024;
constexpr float MIN_T = 0.99e-18f, MAX_T = 1.01e18f;          // T^2 and log2(e) / T are normal f32 values

struct DsP {
    const void* s;            // [R][V] student logits
    const void* tv;           // [R][K] teacher logits
    const void* idx;          // [R][K] int32 / int64
    float* lse;               // [R][2] m = the largest logit, log2 of sum exp((s - m) / T)  (+inf marks a row without a teacher)
    float* loss;              // [R]
    const float* g;           // [R]
    void* ds;
    long R;
    int V, K, tvdt, idx64;
    float c, T;               // c = log2(e) / T
};

__device__ __forceinline__ float tval(const DsP& p, long i) {
    return p.tvdt == PASSION_BF16 ? (float)static_cast<const bf16_t*>(p.tv)[i] : static_cast<const float*>(p.tv)[i];
}
// class of entry i, -1: absent
__device__ __forceinline__ int tidx(const DsP& p, long i) {
    const long v = p.idx64 ? static_cast<const int64_t*>(p.idx)[i] : (long)static_cast<const int32_t*>(p.idx)[i];
    return v >= 0 && v < p.V ? (int)v : -1;
}

// running (reference, sum of exp2(c (s - reference))), s and the reference in the logits' units; -inf references carry an empty sum
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2, float c) {
    const float M = fmaxf(m, m2);
    const float a = M == -INFINITY ? 0.f : M;
    l = l * exp2f((m - a) * c) + l2 * exp2f((m2 - a) * c);
    m = M;
}

template <typename T> __device__ __forceinline__ void vload(const T* p, float* v);
template <> __device__ __forceinline__ void vload<float>(const float* p, float* v) {
    const f32x4 a = load4(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j];
}
template <> __device__ __forceinline__ void vload<bf16_t>(const bf16_t* p, float* v) {
    float t[8];
    VecIO<bf16_t, 8>::load(p, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = t[j];
}
template <typename T> __device__ __forceinline__ void vstore(T* p, const float* v);
template <> __device__ __forceinline__ void vstore<float>(float* p, const float* v) { store4(p, (f32x4){v[0], v[1], v[2], v[3]}); }
template <> __device__ __forceinline__ void vstore<bf16_t>(bf16_t* p, const float* v) {
    typedef float f8 __attribute__((ext_vector_type(8)));
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    *reinterpret_cast<b8*>(p) = __builtin_convertvector((f8){v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}, b8);
}

// N logits into the running pair.  A NaN reaches the sum, whatever the maximum makes of it
template <int N> __device__ __forceinline__ void absorb(const float* v, float c, float& m, float& l) {
    float mx = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) mx = fmaxf(mx, v[j]);
    if (mx > m) { l *= __builtin_amdgcn_exp2f((m - mx) * c); m = mx; }         // m = -inf: l is 0
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += __builtin_amdgcn_exp2f((v[j] - ref) * c);
    l += s;
}

// teacher of one row over the 64 lanes of a wavefront: largest logit and 1 / sum of its softmax; false: no entry
__device__ __forceinline__ bool teacher(const DsP& p, long row, int lane, float& m, float& inv) {
    m = -INFINITY;
    for (int k = lane; k < p.K; k += 64) if (tidx(p, row * p.K + k) >= 0) { const float t = tval(p, row * p.K + k); m = t > m || t != t ? t : m; }
    for (int o = 32; o > 0; o >>= 1) { const float t = __shfl_xor(m, o, 64); m = t > m || t != t ? t : m; }
    if (m == -INFINITY) return false;
    float l = 0.f;
    for (int k = lane; k < p.K; k += 64) if (tidx(p, row * p.K + k) >= 0) l += exp2f((tval(p, row * p.K + k) - m) * p.c);
    l = wave_sum(l);
    inv = 1.f / l;
    return true;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void ds_fwd_row_kernel(DsP p) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float red[2][NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    for (long row = blockIdx.x; row < p.R; row += gridDim.x) {
        const T* s = static_cast<const T*>(p.s) + row * p.V;
        // K <= 64: the first wavefront asks for the teacher's entries and the student's logits at them before the row, and uses them behind it
        const bool early = p.K <= 64 && wv == 0 && lane < p.K;
        int at0 = -1;
        float tv0 = 0.f, z0 = 0.f;
        if (early) {
            at0 = tidx(p, row * p.K + lane);
            tv0 = tval(p, row * p.K + lane);
            z0 = to_f32(s[max(at0, 0)]);
        }
        const int head = (int)min((long)p.V, (long)(((16 - ((uintptr_t)s & 15)) & 15) / sizeof(T)));
        const int nvec = (p.V - head) / VEC, tail = head + nvec * VEC;
        float m = -INFINITY, l = 0.f;
        if (tid < head) { float v = to_f32(s[tid]); absorb<1>(&v, p.c, m, l); }
        if (tid < p.V - tail) { float v = to_f32(s[tail + tid]); absorb<1>(&v, p.c, m, l); }
        int i = tid;
        for (; i + 3 * NT < nvec; i += 4 * NT) {                       // four loads in flight
            float v[4 * VEC];
#pragma unroll
            for (int u = 0; u < 4; ++u) vload<T>(s + head + (long)(i + u * NT) * VEC, v + u * VEC);
            absorb<4 * VEC>(v, p.c, m, l);
        }
        for (; i < nvec; i += NT) {
            float v[VEC];
            vload<T>(s + head + (long)i * VEC, v);
            absorb<VEC>(v, p.c, m, l);
        }
        for (int o = 32; o > 0; o >>= 1) { const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64); join(m, l, m2, l2, p.c); }
        if (lane == 0) { red[0][wv] = m; red[1][wv] = l; }
        __syncthreads();
        if (wv == 0) {
            m = red[0][0]; l = red[1][0];
            for (int w = 1; w < NT / 64; ++w) join(m, l, red[0][w], red[1][w], p.c);
            const float ls = log2f(l);
            float acc = 0.f;
            bool live;
            if (p.K <= 64) {
                const float t = at0 >= 0 ? tv0 : -INFINITY;
                float tm = t;
                for (int o = 32; o > 0; o >>= 1) { const float u = __shfl_xor(tm, o, 64); tm = u > tm || u != u ? u : tm; }
                live = tm != -INFINITY;
                const float d = (t - tm) * p.c, e = live && at0 >= 0 ? exp2f(d) : 0.f, sum = lanes_sum(e, 64), pk = e / sum;
                if (e != 0.f) acc = pk * ((d - log2f(sum)) - ((z0 - m) * p.c - ls));
                acc = lanes_sum(acc, 64);
            } else {
                float tm, inv = 0.f;
                live = teacher(p, row, lane, tm, inv);
                if (live) {
                    const float lt = -log2f(inv);
                    for (int k = lane; k < p.K; k += 64) {
                        const int at = tidx(p, row * p.K + k);
                        if (at < 0) continue;
                        const float d = (tval(p, row * p.K + k) - tm) * p.c, pk = exp2f(d) * inv;
                        if (pk != 0.f) acc += pk * ((d - lt) - ((to_f32(s[at]) - m) * p.c - ls));
                    }
                    acc = wave_sum(acc);
                }
            }
            if (lane == 0) {
                p.loss[row] = live ? p.T * p.T * LN2 * acc : 0.f;
                if (p.lse) {
                    p.lse[2 * row] = m;
                    p.lse[2 * row + 1] = live ? ls : INFINITY;           // +inf marks a row without a teacher (a finite or NaN sum never gives it)
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void ds_bwd_row_kernel(DsP p) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float pk[MAX_K];
    __shared__ int at[MAX_K];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    for (long row = blockIdx.x; row < p.R; row += gridDim.x) {
        const T* s = static_cast<const T*>(p.s) + row * p.V;
        T* o = static_cast<T*>(p.ds) + row * p.V;
        const float m = p.lse[2 * row], ls = p.lse[2 * row + 1], f = p.g[row] * p.T;
        const bool live = ls != INFINITY;
        auto grad = [&](float z) { return f * __builtin_amdgcn_exp2f(__builtin_fmaf(z - m, p.c, -ls)); };        // f q
        if (live && wv == NT / 64 - 1) {                 // the last wavefront, while the others stream the row; read behind the barrier below
            float tm, inv = 0.f;
            teacher(p, row, lane, tm, inv);
            for (int k = lane; k < p.K; k += 64) {
                at[k] = tidx(p, row * p.K + k);
                pk[k] = at[k] < 0 ? 0.f : exp2f((tval(p, row * p.K + k) - tm) * p.c) * inv;
            }
        }
        // the student's and the gradient's rows start at the same offset from a 16-byte point (both bases are aligned)
        const int head = (int)min((long)p.V, (long)(((16 - ((uintptr_t)s & 15)) & 15) / sizeof(T)));
        const int nvec = (p.V - head) / VEC, tail = head + nvec * VEC;
        if (live) {
            if (tid < head) o[tid] = from_f32<T>(grad(to_f32(s[tid])));
            if (tid < p.V - tail) o[tail + tid] = from_f32<T>(grad(to_f32(s[tail + tid])));
            int i = tid;
            for (; i + 3 * NT < nvec; i += 4 * NT) {
                float v[4][VEC];
#pragma unroll
                for (int u = 0; u < 4; ++u) vload<T>(s + head + (long)(i + u * NT) * VEC, v[u]);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[u][j] = grad(v[u][j]);
                    vstore<T>(o + head + (long)(i + u * NT) * VEC, v[u]);
                }
            }
            for (; i < nvec; i += NT) {
                float v[VEC];
                vload<T>(s + head + (long)i * VEC, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = grad(v[j]);
                vstore<T>(o + head + (long)i * VEC, v);
            }
            stores_done();                               // the row is written before the named classes are written again
        } else {
            const float z[VEC] = {};
            if (tid < head) o[tid] = from_f32<T>(0.f);
            if (tid < p.V - tail) o[tail + tid] = from_f32<T>(0.f);
            for (int i = tid; i < nvec; i += NT) vstore<T>(o + head + (long)i * VEC, z);
        }
        __syncthreads();
        if (live)
            for (int k = tid; k < p.K; k += NT) {
                const int a = at[k];
                if (a < 0) continue;
                float sum = 0.f;
                bool first = true;
                for (int j = 0; j < p.K; ++j)
                    if (at[j] == a) { sum += pk[j]; first &= j >= k; }
                if (first) o[a] = from_f32<T>(f * (__builtin_amdgcn_exp2f(__builtin_fmaf(to_f32(s[a]) - m, p.c, -ls)) - sum));
            }
        __syncthreads();
    }
}

// V <= 512: G lanes a row, 8 classes a lane (4 where V <= 4): class of element j: VPT lane + j (VEC: rows of whole aligned vectors) or j G + lane
template <typename T, int VPT, bool VEC, bool BWD>
__global__ __launch_bounds__(256) void ds_small_kernel(DsP p, int G) {
    const int t = threadIdx.x & (G - 1);
    const long row0 = (long)blockIdx.x * (256 / G) + threadIdx.x / G, step = (long)gridDim.x * (256 / G);
    for (long r = row0; r - threadIdx.x / G < p.R; r += step) {          // whole wavefronts stay together (shuffles)
        const bool ok = r < p.R;
        const long row = ok ? r : p.R - 1;
        const T* s = static_cast<const T*>(p.s) + row * p.V;
        float x[VPT];
        if (VEC && t * VPT < p.V) {
            if constexpr (VPT * sizeof(T) >= 16) {
#pragma unroll
                for (int u = 0; u < VPT * (int)sizeof(T) / 16; ++u) vload<T>(s + t * VPT + u * (16 / (int)sizeof(T)), x + u * (16 / (int)sizeof(T)));
            } else {
                const f32x4 a = load4(s + t * VPT);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = a[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) { const int c = VEC ? t * VPT + j : j * G + t; x[j] = c < p.V ? to_f32(s[c]) : -INFINITY; }
        }
        // teacher
        float tm = -INFINITY;
        for (int k = t; k < p.K; k += G) if (tidx(p, row * p.K + k) >= 0) { const float v = tval(p, row * p.K + k); tm = v > tm || v != v ? v : tm; }
        for (int o = G >> 1; o > 0; o >>= 1) { const float v = __shfl_xor(tm, o, 64); tm = v > tm || v != v ? v : tm; }
        const bool live = tm != -INFINITY;
        float tl = 0.f;
        if (live) for (int k = t; k < p.K; k += G) if (tidx(p, row * p.K + k) >= 0) tl += exp2f((tval(p, row * p.K + k) - tm) * p.c);
        for (int o = G >> 1; o > 0; o >>= 1) tl += __shfl_xor(tl, o, 64);
        const float inv = 1.f / tl;
        if constexpr (!BWD) {
            float m = -INFINITY, l = 0.f;
            absorb<VPT>(x, p.c, m, l);
            for (int o = G >> 1; o > 0; o >>= 1) { const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64); join(m, l, m2, l2, p.c); }
            const float ls = log2f(l);
            float acc = 0.f;
            if (live) {
                const float lt = log2f(tl);
                for (int k = t; k < p.K; k += G) {
                    const int a = tidx(p, row * p.K + k);
                    if (a < 0) continue;
                    const float d = (tval(p, row * p.K + k) - tm) * p.c, pk = exp2f(d) * inv;
                    if (pk != 0.f) acc += pk * ((d - lt) - ((to_f32(s[a]) - m) * p.c - ls));
                }
            }
            for (int o = G >> 1; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
            if (ok && t == 0) {
                p.loss[row] = live ? p.T * p.T * LN2 * acc : 0.f;
                if (p.lse) { p.lse[2 * row] = m; p.lse[2 * row + 1] = ls; }
            }
        } else {
            const float m = p.lse[2 * row], ls = p.lse[2 * row + 1], f = p.g[row] * p.T;
#pragma unroll
            for (int j = 0; j < VPT; ++j) x[j] = live ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[j] - m, p.c, -ls)) : 0.f;
            if (live)
                for (int k = 0; k < p.K; ++k) {
                    const int a = tidx(p, row * p.K + k);
                    if (a < 0) continue;
                    const float pk = exp2f((tval(p, row * p.K + k) - tm) * p.c) * inv;
#pragma unroll
                    for (int j = 0; j < VPT; ++j) x[j] -= (VEC ? t * VPT + j : j * G + t) == a ? pk : 0.f;
                }
#pragma unroll
            for (int j = 0; j < VPT; ++j) x[j] = live ? x[j] * f : 0.f;
            T* o = static_cast<T*>(p.ds) + row * p.V;
            if (ok) {
                if (VEC && t * VPT < p.V) {
                    if constexpr (VPT * sizeof(T) >= 16) {
#pragma unroll
                        for (int u = 0; u < VPT * (int)sizeof(T) / 16; ++u) vstore<T>(o + t * VPT + u * (16 / (int)sizeof(T)), x + u * (16 / (int)sizeof(T)));
                    } else store4(o + t * VPT, (f32x4){x[0], x[1], x[2], x[3]});
                } else {
#pragma unroll
                    for (int j = 0; j < VPT; ++j) { const int c = VEC ? t * VPT + j : j * G + t; if (c < p.V) o[c] = from_f32<T>(x[j]); }
                }
            }
        }
    }
}

template <typename T, bool BWD>
int launch(const DsP& p, hipStream_t st) {
    const bool aligned = !(((uintptr_t)p.s | (uintptr_t)p.ds) & 15);
    if (p.V <= SMALL_V) {
        const int vpt = p.V <= 4 ? 4 : 8;
        int G = 1;
        while (G * vpt < p.V) G *= 2;
        const bool vec = aligned && p.V % vpt == 0;
        const long want = (p.R + 256 / G - 1) / (256 / G);
        const dim3 grid((unsigned)hmin(want, 1L << 20));
        if (vpt == 4) {
            if (vec) hipLaunchKernelGGL((ds_small_kernel<T, 4, true, BWD>), grid, dim3(256), 0, st, p, G);
            else hipLaunchKernelGGL((ds_small_kernel<T, 4, false, BWD>), grid, dim3(256), 0, st, p, G);
        } else {
            if (vec) hipLaunchKernelGGL((ds_small_kernel<T, 8, true, BWD>), grid, dim3(256), 0, st, p, G);
            else hipLaunchKernelGGL((ds_small_kernel<T, 8, false, BWD>), grid, dim3(256), 0, st, p, G);
        }
    } else {
        if (BWD && !aligned) return -1005;
        // few long rows: 1024 threads a row keep the whole row in flight; many rows: 256 threads, several rows a CU.  bf16, K = 8, with the gradient, 1024 / 256 threads: 64 x 32001 13.7 / 14.2 us,
        // 256 x 130000 39.6 / 42.0, 2000 x 32001 109 / 72.  Between (more rows than CUs, fewer than 1024) 256 are faster already: 512 x 32001 32.6 / 23.1, 1000 x 32001 60 / 38.5
        const bool wide = p.R < 1024 && p.V >= 4096;
        const dim3 grid((unsigned)hmin(p.R, 1L << 20));
        if (BWD) {
            if (wide) hipLaunchKernelGGL((ds_bwd_row_kernel<T, 1024>), grid, dim3(1024), 0, st, p);
            else hipLaunchKernelGGL((ds_bwd_row_kernel<T, 256>), grid, dim3(256), 0, st, p);
        } else {
            if (wide) hipLaunchKernelGGL((ds_fwd_row_kernel<T, 1024>), grid, dim3(1024), 0, st, p);
            else hipLaunchKernelGGL((ds_fwd_row_kernel<T, 256>), grid, dim3(256), 0, st, p);
        }
    }
    LAUNCH_RET();
    return 0;
}

bool bad(int64_t R, int V, int K, float T, int dt, int tvdt) {
    return R < 1 || V < 1 || K < 1 || K > MAX_K || !(T >= MIN_T && T <= MAX_T) || (dt != PASSION_F32 && dt != PASSION_BF16) || (tvdt != PASSION_F32 && tvdt != PASSION_BF16);
}

}  // namespace

extern "C" int passion_topk_distill_max_k(void) { return MAX_K; }

extern "C" int passion_topk_distill_fwd(const void* logits, int dtype, const void* values, int values_dtype, const void* index, int index64, int64_t R, int V, int K,
                                        float temp, float* loss, float* lse, void* stream) {
    if (bad(R, V, K, temp, dtype, values_dtype) || !logits || !values || !index || !loss) return -1003;
    DsP p{};
    p.s = logits; p.tv = values; p.idx = index; p.lse = lse; p.loss = loss; p.R = R; p.V = V; p.K = K; p.tvdt = values_dtype; p.idx64 = index64;
    p.c = LOG2E / temp; p.T = temp;
    return dtype == PASSION_F32 ? launch<float, false>(p, (hipStream_t)stream) : launch<bf16_t, false>(p, (hipStream_t)stream);
}

extern "C" int passion_topk_distill_bwd(const void* logits, int dtype, const void* values, int values_dtype, const void* index, int index64, int64_t R, int V, int K,
                                        float temp, const float* lse, const float* dloss, void* dlogits, void* stream) {
    if (bad(R, V, K, temp, dtype, values_dtype) || !logits || !values || !index || !lse || !dloss || !dlogits) return -1003;
    DsP p{};
    p.s = logits; p.tv = values; p.idx = index; p.lse = const_cast<float*>(lse); p.g = dloss; p.ds = dlogits; p.R = R; p.V = V; p.K = K;
    p.tvdt = values_dtype; p.idx64 = index64; p.c = LOG2E / temp; p.T = temp;
    return dtype == PASSION_F32 ? launch<float, true>(p, (hipStream_t)stream) : launch<bf16_t, true>(p, (hipStream_t)stream);
}
