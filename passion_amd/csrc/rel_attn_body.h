// Kernels of attention with a learned relative position bias (host side and the mathematics: rel_attn.hip).  Included once per tensor type.
//
// Score tiles as in flash_attn.hip: S^T[key][q] = K . Q^T with 32x32 matrix instructions, a lane owns one query (column l & 31) and 16 of the
// tile's 32 keys (rows (r & 3) + 8 (r >> 2) + 4 (l >> 5)), so a row's maximum and sum are in registers plus one exchange with lane l ^ 32, and
// the probabilities are the B operand of the next product where they stand.  The key-major kernel is the mirror image.
//   bf16: v_mfma_f32_32x32x16_bf16, 16 bytes of a row a lane and instruction; transposed operands by ds_read_b64_tr_b16.
//   f32:  v_mfma_f32_32x32x2_f32, four instructions per 16 bytes (the four k pairs a lane's 16 bytes hold); accumulator register r as the B
//         operand of one instruction, whose A operand is a plain b32 read of image row (r & 3) + 8 (r >> 2) + 4 (l >> 5).  Full f32 products.
//
// Bias of a pair, in log2 units, by its offset o(i, j) = pos(i) - pos(j) + const:
//   BOX    the head's whole expanded table in LDS (up to 4096 offsets: grids up to 8 x 8 x 8 and a little beyond), one LDS read a score;
//   LINE   a 1D raster: the offsets of a (query tile, key block) pair are one window of 32 NW + BLK - 1 values, staged with the block, and the LDS
//          address of a score is a lane constant plus an immediate;
//   GATHER one global read a score (L1 / L2), any grid.
// Gradient of the table: sums of dS by offset, without atomics and in a fixed order.
//   LINE: in the key-major kernel.  A wavefront's 32 keys x 32 queries of dS go through LDS as [key][query] and are read back along the diagonals: row kk at
//         column lane - 32 + kk (zeros on either side of a row), so a lane's values belong to one offset: an LDS read with an immediate address and an add each,
//         conflict-free.  The 32 offsets that no later tile of queries reaches leave for a slab row of the key tile in one aligned store; the rest move on.
//         (LDS float atomics into a window instead took 170 to 280 cycles an instruction: 3.2 ms over 8000 x 8000 x 8 heads of 128, where this kernel and the
//         fold of its sums now take 0.85.)
//   BOX, GATHER: a kernel of its own sums dS over batch and repeated cells for every pair of cells (a pair's bias is loaded once, its sum stays in a
//         register), and the sums by offset follow from that dense matrix.
#include "common.h"
#include "passion_hip.h"
#include "rel_attn.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float LAZY = 8.0f;           // log2 units by which a block must exceed the running reference before it moves
enum { NONE = 0, BOX = 1, LINE = 2, GATHER = 3 };

template <typename T> constexpr int blk() { return sizeof(T) == 2 ? 64 : 32; }                       // rows staged a step

// LDS images: rows of DP elements without padding, the 16-byte chunks of a row permuted by its number (chunk c of row r lies at place c ^ swz(r)), so that both ways of
// reading are free of bank conflicts: 16 rows at one column (row fragments: 16 places), and 64 bytes of 4 consecutive rows (transposed fragments: 4 windows).  (Rows
// padded by 16 bytes for the first way met 2- to 4-way conflicts the second way.)
template <int BYTES> __device__ __forceinline__ int swz(int row) {
    if constexpr (BYTES >= 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (BYTES == 128) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int j = 0; j < 16; ++j) z[j] = 0.f;
    return z;
}
__device__ __forceinline__ float half_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// acc += A . B over the k range of one 16-byte chunk a lane
template <typename T> __device__ __forceinline__ f32x16 dot(u32x4 a, u32x4 b, f32x16 acc) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    else {
#pragma unroll
        for (int t = 0; t < 4; ++t) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[t]), __uint_as_float(b[t]), acc, 0, 0, 0);
        return acc;
    }
}
// out[dt] += (image rows r0 .. r0 + 31, columns 32 dt ..)^T . acc, acc an accumulator tile whose rows are those image rows (r0 a multiple of 32).  AHEAD: the image's
// fragments are requested by load(), ahead of the arithmetic that forms acc; else by product() as it goes (kernels that have no registers left; f32)
template <typename T, int DP, bool AHEAD> struct TrFrags {
    static constexpr int ND = DP / 32, STRIDE = DP * (int)sizeof(T);
    bf16x8 a[AHEAD ? 2 : 1][AHEAD ? ND : 1];
    const char* base;
    int q4, x;
    __device__ __forceinline__ bf16x8 frag(int s, int dt, int lane) const {
        s16x4 part[2];
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
            // row 16 s + 8 hi + 4 h + q4, chunk 4 dt + x: its place from swz() of that row
            const int grp = STRIDE == 256 ? dt ^ q4 : STRIDE == 128 ? dt ^ (q4 >> 1) : 0;
            const char* p = base + (16 * s + 8 * hi) * STRIDE + (grp << 6) + ((x ^ (2 * hi)) << 4);
            part[hi] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p));
        }
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void load(const char* img, int r0, int lane) {
        if constexpr (sizeof(T) == 2) {
            const int n = lane & 15, g = lane >> 4, h = g >> 1, pq = n & 3;
            q4 = n >> 2;
            x = (2 * (g & 1) + (pq >> 1)) ^ h;
            base = img + (r0 + 4 * h + q4) * STRIDE + (pq & 1) * 8;
            if constexpr (AHEAD) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) a[s][dt] = frag(s, dt, lane);
            }
        } else base = img + (r0 + 4 * (lane >> 5)) * STRIDE;
    }
    __device__ __forceinline__ void product(const f32x16& acc, f32x16 (&out)[ND], int lane) const {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 b;
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = (__bf16)acc[8 * s + j];
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    bf16x8 f;
                    if constexpr (AHEAD) f = a[s][dt];
                    else f = frag(s, dt, lane);
                    out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, b, out[dt], 0, 0, 0);
                }
            }
        } else {
            const int h = lane >> 5, col = lane & 31;
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    const int row = (r & 3) + 8 * (r >> 2) + 4 * h, c = 8 * dt + (col >> 2);
                    const float v = *reinterpret_cast<const float*>(base + ((r & 3) + 8 * (r >> 2)) * STRIDE + ((c ^ swz<STRIDE>(row)) << 4) + (col & 3) * 4);
                    out[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, acc[r], out[dt], 0, 0, 0);
                }
        }
    }
};
// the row fragments of image rows r0 .. r0 + 31 (lane: row r0 + (l & 31), half l >> 5 of every 32 bytes)
template <typename T, int DP> struct RowFrags {
    static constexpr int STRIDE = DP * (int)sizeof(T), N = STRIDE / 32;
    u32x4 a[N];
    __device__ __forceinline__ void load(const char* img, int r0, int lane) {
        const char* row = img + (r0 + (lane & 31)) * STRIDE;
        const int at = ((lane >> 5) ^ swz<STRIDE>(lane & 31)) << 4;
#pragma unroll
        for (int s = 0; s < N; ++s) a[s] = *reinterpret_cast<const u32x4*>(row + ((32 * s) ^ at));
    }
    __device__ __forceinline__ f32x16 times(const u32x4 (&b)[N], f32x16 acc) const {
#pragma unroll
        for (int s = 0; s < N; ++s) acc = dot<T>(a[s], b[s], acc);
        return acc;
    }
};

// a tile of BLK rows x DP columns in registers, NT threads, on its way to LDS.  Loads are unconditional (rows past `last` read row `last`, columns past D read
// column 0) from a uniform base with 32-bit lane offsets; what is not there becomes 0 when it is stored
template <typename T, int DP, int NT> struct Tile {
    static constexpr int CPR = DP * (int)sizeof(T) / 16, N = blk<T>() * CPR / NT, STEP = NT / CPR;
    u32x4 r[N];
    __device__ __forceinline__ void fetch(const T* base, int stride, int last, int D, int tid) {      // stride in bytes (64 rows stay below 2^31: checked by the host)
        const int row = tid / CPR, c = (tid % CPR) * 16;
        const unsigned col = c < D * (int)sizeof(T) ? c : 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            r[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) + ((unsigned)min(row + i * STEP, last) * (unsigned)stride + col));
    }
    __device__ __forceinline__ void commit(char* img, int tid, uint64_t valid, int D) const {
        constexpr int STRIDE = DP * (int)sizeof(T);
        const int row = tid / CPR, c = tid % CPR;
        const bool whole = valid == all_rows() && D == DP, in = c * 16 < D * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = row + i * STEP;
            u32x4 v = r[i];
            if (!whole) v = in && row_bit(valid, row, i * STEP) ? v : (u32x4){0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4*>(img + at * STRIDE + ((c ^ swz<STRIDE>(at)) << 4)) = v;
        }
    }
    // bit row + add of a block's rows.  In 32 bits on purpose: a 64-bit vector shift whose amount the compiler has put into the last register that the wavefront
    // owns (v255 here) reads another register's value instead, in every wavefront but a SIMD's first, and a valid row was then stored as zeros
    static __device__ __forceinline__ bool row_bit(uint64_t valid, int row, int add) {
        const uint32_t lo = (uint32_t)valid, hi = (uint32_t)(valid >> 32);
        if constexpr (STEP <= 32) return ((add < 32 ? lo : hi) >> (row + (add & 31))) & 1;
        else return ((row < 32 ? lo : hi) >> (row & 31)) & 1;      // all 64 rows at once: add is 0
    }
    static __device__ __forceinline__ constexpr uint64_t all_rows() { return blk<T>() == 64 ? ~0ull : 0xffffffffull; }
};
// what the rounding of dS to a bf16 operand leaves.  In bf16 the probabilities (for out and dV) and dS (for dQ and dK) are rounded once to the matrix operand's type, as much as the
// result itself is: out, dV, dQ and dK are off by 2.3 to 2.4e-3 of their norm where the rounding of the result alone is 1.7e-3.  Heads up to 32 wide add the product of dS's
// rest, which brings dQ and dK to 1.7e-3 (4000^2, 8 heads of 32: forward + backward 339 us instead of 311).  For wider ones it was measured and left: dQ and dK at 1.7e-3 as well, but
// 1D 2000^2, 8 heads of 64: dQ 31 -> 35 us, dK / dV 53 -> 69 (no registers left); 8000^2, 8 heads of 128 on 4: 1690 -> 1815 us in all
__device__ __forceinline__ f32x16 rest(const f32x16& a) {
    f32x16 r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = a[i] - (float)(bf16_t)a[i];
    return r;
}
// bits of the first n rows of a block
__device__ __forceinline__ uint64_t first_rows(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// place of token t in the box of offsets (before the constant that makes differences non-negative)
__device__ __forceinline__ int place(const RelP& p, int t) {
    t %= p.vol;
    const int z = t / (p.gh * p.gw), yx = t - z * (p.gh * p.gw), y = yx / p.gw, x = yx - y * p.gw;
    return (z * (2 * p.gh - 1) + y) * (2 * p.gw - 1) + x;
}
// GATHER: bias of head `head` at offset o: the expanded table, or (few queries: no expansion pass) the table itself
__device__ __forceinline__ float gather_bias(const RelP& p, int head, int o) {
    if (p.e) return p.e[(long)head * p.nd + o];
    return rel_log2_bias(p.table, p.tdt, p.buckets ? p.buckets[o] : o, p.nb, head, p.H);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// query-major: MODE 0 forward (out, lse or split partials), MODE 1 backward (dQ; delta corrected in place).
// grid (ceil(rows / (32 NW)) * nsplit, heads, B).  pack (forward, few queries): a workgroup's rows are the Nq queries of all the heads that
// share a key / value head, so that K and V are read once for them
template <typename T, int DP, int NW, int MODE, int BIAS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 || (DP == 128 && NW == 1) ? 1 : 2))) void rel_q_kernel(RelP p) {
    constexpr int NT = 64 * NW, BLKN = blk<T>(), KT = BLKN / 32, NCH = DP * (int)sizeof(T) / 32, ND = DP / 32;
    constexpr int KIMG = BLKN * DP * (int)sizeof(T), VIMG = KIMG, POS = BLKN * 4, WIN = (32 * NW + BLKN) * 4;
    constexpr bool AHEAD = sizeof(T) == 2 && DP <= 64;              // fragments requested ahead: where 256 registers hold them
    // few queries (LINE): a window a head of the tile, BLK + Nq values each
    const int wrow = BLKN + p.Nq, BUF = KIMG + VIMG + (BIAS == LINE ? (p.few ? (p.pack ? p.H / p.Hkv : 1) * wrow * 4 + 15 & ~15 : WIN) : BIAS == NONE ? 0 : POS);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = lane >> 5;
    const int b = blockIdx.z, rep = p.H / p.Hkv;
    const int split = blockIdx.x % p.nsplit, tile = blockIdx.x / p.nsplit;
    const int rows = p.pack ? p.Nq * rep : p.Nq;
    const int row = (tile * NW + wv) * 32 + (lane & 31);
    const bool qok = row < rows;
    const int rowc = qok ? row : rows - 1;
    const int head = p.pack ? blockIdx.y * rep + rowc / p.Nq : blockIdx.y, qi = p.pack ? rowc % p.Nq : rowc;
    const int hk = p.pack ? blockIdx.y : blockIdx.y / rep;
    const T* kb_ = static_cast<const T*>(p.k) + (long)b * p.ks[0] + (long)hk * p.ks[2];
    const T* vb_ = static_cast<const T*>(p.v) + (long)b * p.vs[0] + (long)hk * p.vs[2];
    const int nblk_all = (p.Nk + BLKN - 1) / BLKN;
    const int kb0 = (int)((long)split * nblk_all / p.nsplit), kb1 = (int)((long)(split + 1) * nblk_all / p.nsplit);
    const long orow = ((long)b * p.Nq + qi) * p.H + head, lrow = ((long)b * p.H + head) * p.Nq + qi;

    u32x4 qf[NCH], df[NCH];
    {
        const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(p.q) + (long)b * p.qs[0] + (long)qi * p.qs[1] + (long)head * p.qs[2]);
        const char* dp = MODE == 1 ? reinterpret_cast<const char*>(static_cast<const T*>(p.dout) + orow * p.D) : nullptr;
#pragma unroll
        for (int s = 0; s < NCH; ++s) {
            const bool in = qok && (32 * s + 16 * h) < p.D * (int)sizeof(T);
            qf[s] = (u32x4){0u, 0u, 0u, 0u};
            if (in) qf[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s + 16 * h);
            if (MODE == 1) {
                df[s] = (u32x4){0u, 0u, 0u, 0u};
                if (in) df[s] = *reinterpret_cast<const u32x4*>(dp + 32 * s + 16 * h);
            }
        }
    }
    float lse2 = INFINITY, dlt = 0.f;                       // no such query: p = exp2(. - inf) = 0
    if (MODE == 1 && qok) { lse2 = p.lse[lrow]; dlt = p.delta[lrow]; }
    const int aq = (BIAS == BOX || BIAS == GATHER) ? place(p, p.q0 + qi) + p.omax : 0;      // offset of a pair = aq - place(key)

    float* tab = reinterpret_cast<float*>(lds + 2 * BUF);                                  // BOX: the head's table behind the two buffers
    if (BIAS == BOX)
        for (int i = tid; i < p.nd; i += NT) tab[i] = p.e[(long)blockIdx.y * p.nd + i];
    const bool wave_on = tile * NW + wv < (rows + 31) / 32;       // a wavefront without a row stages tiles and keeps out of the rest

    f32x16 o[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = zero16();
    float l_run = 0.f, m_run = -INFINITY;               // backward: l_run sums dS

    Tile<T, DP, NT> kt_, vt_;
    uint64_t valid = 0, vnext = 0;
    bool there = false;                                        // this lane's key of the block on its way takes part
    constexpr int NWIN = (32 * NW + BLKN + NT - 1) / NT;
    float win[BIAS == LINE ? NWIN : 1];
    int kpos = 0;
    // (width 128: the value tile follows the key tile through the same registers, half a step later)
    constexpr bool HALVES = sizeof(T) == 2 && DP == 128;
    auto fetch_v = [&](int kb) {
        const int key0 = kb * BLKN, last = min(p.Nk - 1 - key0, BLKN - 1);
        vt_.fetch(vb_ + key0 * p.vs[1], (int)(p.vs[1] * sizeof(T)), last, p.D, tid);
    };
    auto fetch = [&](int kb) {
        const int key0 = kb * BLKN, last = min(p.Nk - 1 - key0, BLKN - 1);
        kt_.fetch(kb_ + key0 * p.ks[1], (int)(p.ks[1] * sizeof(T)), last, p.D, tid);
        if (!HALVES) fetch_v(kb);
        there = lane <= last;
        if (p.mask) there = there && p.mask[(long)b * p.Nk + key0 + min(lane, last)];
        if (BIAS == LINE && p.few) {                       // straight into the next buffer (last read before the previous barrier), from the table itself
            float* w = reinterpret_cast<float*>(lds + ((kb - kb0) & 1) * BUF + KIMG + VIMG);
            const int first = p.q0 - (kb * BLKN + BLKN - 1) + p.gw - 1, heads = p.pack ? rep : 1;
            for (int i = tid; i < wrow; i += NT) {
                const int at = first + i;
                const bool in = at >= 0 && at < p.nd;
                const int c = in ? (p.buckets ? p.buckets[at] : at) : -1;
                for (int g = 0; g < heads; ++g) w[g * wrow + i] = rel_log2_bias(p.table, p.tdt, c, p.nb, blockIdx.y * heads + g, p.H);
            }
        } else if (BIAS == LINE) {
            // window value w <-> offset of (query tile 0 of the workgroup, last key of the block) + w
            const int first = p.q0 + tile * NW * 32 - (kb * BLKN + BLKN - 1) + p.gw - 1;
#pragma unroll
            for (int i = 0; i < NWIN; ++i) {
                const int at = first + i * NT + tid;
                win[i] = (i * NT + tid < 32 * NW + BLKN && at >= 0 && at < p.nd) ? p.e[(long)blockIdx.y * p.nd + at] : 0.f;
            }
        }
        if ((BIAS == BOX || BIAS == GATHER) && tid < BLKN) kpos = place(p, min(kb * BLKN + tid, p.Nk - 1));
    };
    auto commit_k = [&](char* buf) {
        vnext = __ballot(there);                               // lanes hold a key each (BLK = 32: the upper half none: last < 32)
        kt_.commit(buf, tid, vnext, p.D);
    };
    auto commit = [&](char* buf) {
        if (!HALVES) commit_k(buf);
        vt_.commit(buf + KIMG, tid, vnext, p.D);
        if (BIAS == LINE && !p.few) {
#pragma unroll
            for (int i = 0; i < NWIN; ++i)
                if (i * NT + tid < 32 * NW + BLKN) reinterpret_cast<float*>(buf + KIMG + VIMG)[i * NT + tid] = win[i];
        }
        if ((BIAS == BOX || BIAS == GATHER) && tid < BLKN) reinterpret_cast<int*>(buf + KIMG + VIMG)[tid] = kpos;
    };
    auto step = [&](int kb, auto between) {
        const char* kimg = lds + ((kb - kb0) & 1) * BUF;
        const char* vimg = kimg + KIMG;
        if (!(valid && wave_on)) between();
        else {
            // scores of 32 keys in log2 units: scale * log2(e) * s + bias, -inf where the key does not take part
            const float* wl = reinterpret_cast<const float*>(vimg + VIMG) + (p.few ? (p.pack ? rowc / p.Nq : 0) * wrow + qi : 32 * wv + (lane & 31)) + BLKN - 1 - 4 * h;
            const bool full = valid == Tile<T, DP, NT>::all_rows();
            const uint64_t vh = h ? valid >> 4 : valid;      // (constant shifts: see row_bit)
            auto bias_of = [&](int kt) {                        // requested together, ahead of the products where registers allow
                f32x16 e = zero16();
                if (BIAS == NONE) return e;
                int4 kp[4];
                if (BIAS == BOX || BIAS == GATHER) {
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) kp[g4] = *reinterpret_cast<const int4*>(vimg + VIMG + (kt * 32 + 8 * g4 + 4 * h) * 4);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int g4 = r >> 2, j = r & 3;
                    if (BIAS == LINE) e[r] = wl[-(kt * 32 + 8 * g4 + j)];
                    else {
                        const int off = aq - (j == 0 ? kp[g4].x : j == 1 ? kp[g4].y : j == 2 ? kp[g4].z : kp[g4].w);
                        e[r] = BIAS == BOX ? tab[off] : gather_bias(p, head, off);
                    }
                }
                return e;
            };
            auto finish = [&](f32x16 st, f32x16 e, int kt) {
#pragma unroll
                for (int r = 0; r < 16; ++r) st[r] = BIAS == NONE ? st[r] * p.c : __builtin_fmaf(st[r], p.c, e[r]);
                if (!full) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!((vh >> (kt * 32 + (r & 3) + 8 * (r >> 2))) & 1)) st[r] = -INFINITY;
                }
                return st;
            };
            if (MODE == 0) {
                f32x16 st[KT];
                RowFrags<T, DP> kf[KT];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) kf[kt].load(kimg, kt * 32, lane);
                f32x16 e[KT];
                if (AHEAD) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) e[kt] = bias_of(kt);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) st[kt] = kf[kt].times(qf, zero16());
                between();
                TrFrags<T, DP, AHEAD> vf[KT];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) vf[kt].load(vimg, kt * 32, lane);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    if (!AHEAD) {
                        e[kt] = bias_of(kt);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    st[kt] = finish(st[kt], e[kt], kt);
                }
                float mx = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[kt][r]);
                mx = half_max(mx);
                const bool move = mx > m_run + LAZY;                              // first key of a row: m_run = -inf
                if (__any(move)) {
                    const float m_new = move ? mx : m_run;
                    const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
                }
                const float ref = m_run == -INFINITY ? 0.f : m_run;                // nothing left of the row so far: exp2(-inf - 0) = 0
                float psum = 0.f;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        st[kt][r] = __builtin_amdgcn_exp2f(st[kt][r] - ref);
                        psum += st[kt][r];
                    }
                l_run += psum;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) vf[kt].product(st[kt], o, lane);
            } else {
                // a row of dS sums to 0; what it sums to instead is the error of delta, which was formed from the rounded out.  One block of keys (few keys: there it
                // shows): measured first and taken off; else by the kernels that follow, through the corrected delta
                // scores and dP - delta (delta is where the product starts from)
                auto tile = [&](int kt, f32x16& st, f32x16& dp) {
                    RowFrags<T, DP> kf, vf;
                    kf.load(kimg, kt * 32, lane);
                    if (AHEAD) {
                        vf.load(vimg, kt * 32, lane);
                        const f32x16 e = bias_of(kt);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int r = 0; r < 16; ++r) dp[r] = -dlt;
                        st = kf.times(qf, zero16());
                        dp = vf.times(df, dp);
                        st = finish(st, e, kt);
                    } else {                                    // (apart, so that no more than one product's fragments are held)
                        st = kf.times(qf, zero16());
                        __builtin_amdgcn_sched_barrier(0);
                        vf.load(vimg, kt * 32, lane);
#pragma unroll
                        for (int r = 0; r < 16; ++r) dp[r] = -dlt;
                        dp = vf.times(df, dp);
                        __builtin_amdgcn_sched_barrier(0);
                        st = finish(st, bias_of(kt), kt);
                    }
                };
                if (nblk_all == 1) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        f32x16 st, dp;
                        tile(kt, st, dp);
#pragma unroll
                        for (int r = 0; r < 16; ++r) l_run = __builtin_fmaf(__builtin_amdgcn_exp2f(st[r] - lse2), dp[r], l_run);
                    }
                    dlt += half_sum(l_run);
                    l_run = 0.f;
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    f32x16 st, dp;
                    tile(kt, st, dp);
                    TrFrags<T, DP, AHEAD> kt2;
                    kt2.load(kimg, kt * 32, lane);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        dp[r] *= __builtin_amdgcn_exp2f(st[r] - lse2);
                        l_run += dp[r];
                    }
                    kt2.product(dp, o, lane);
                    if constexpr (sizeof(T) == 2 && DP == 32) kt2.product(rest(dp), o, lane);
                    if (kt == 0) between();
                }
            }
        }
    };
    // (the last block apart: a load that may or may not be waited for later costs a wait for everything at the loop's top)
    if (kb0 < kb1) {
        fetch(kb0);
        if (HALVES) { commit_k(lds); fetch_v(kb0); }
        commit(lds);
        valid = vnext;
        __syncthreads();
        for (int kb = kb0; kb + 1 < kb1; ++kb) {
            char* next = lds + ((kb + 1 - kb0) & 1) * BUF;
            fetch(kb + 1);
            step(kb, [&] {
                if (HALVES) { commit_k(next); fetch_v(kb + 1); }
            });
            commit(next);
            valid = vnext;
            __syncthreads();
        }
        step(kb1 - 1, [] {});
    }

    if (MODE == 0) {
        const float l = half_sum(l_run);
        if (p.nsplit > 1) {
            if (qok) {
                const long at = (long)split * p.B * p.H * p.Nq + lrow;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const int d = dt * 32 + 8 * g4 + 4 * h;
                        if (d < p.D) store4(p.po + at * p.D + d, (f32x4){o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]});
                    }
                if (h == 0) { p.pm[at] = m_run; p.pl[at] = l; }
            }
            return;
        }
        if (qok) {
            const float f = l == 0.f ? 0.f : 1.f / l;                              // a row without a key: 0
            T* dst = static_cast<T*>(p.out) + orow * p.D;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int d = dt * 32 + 8 * g4 + 4 * h;
                    if (d < p.D) store4(dst + d, (f32x4){o[dt][4 * g4] * f, o[dt][4 * g4 + 1] * f, o[dt][4 * g4 + 2] * f, o[dt][4 * g4 + 3] * f});
                }
            if (h == 0 && p.lse) p.lse[lrow] = l == 0.f ? INFINITY : m_run + __builtin_amdgcn_logf(l);
        }
    } else if (p.nsplit > 1) {                                                    // joined afterwards, delta's correction with it
        const float off = half_sum(l_run);
        if (qok) {
            const long at = (long)split * p.B * p.H * p.Nq + lrow;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int d = dt * 32 + 8 * g4 + 4 * h;
                    if (d < p.D) store4(p.po + at * p.D + d, (f32x4){o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]});
                }
            if (h == 0) p.pm[at] = off;
        }
    } else {
        if (qok) {
            T* dst = static_cast<T*>(p.dq) + orow * p.D;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int d = dt * 32 + 8 * g4 + 4 * h;
                    if (d < p.D)
                        store4(dst + d, (f32x4){o[dt][4 * g4] * p.scale, o[dt][4 * g4 + 1] * p.scale, o[dt][4 * g4 + 2] * p.scale, o[dt][4 * g4 + 3] * p.scale});
                }
        }
        const float off = half_sum(l_run);
        if (qok && h == 0) p.delta[lrow] = dlt + off;
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// key-major backward: dK, dV.  grid (ceil(Nk / (32 NW)) * ksplit, Hkv, B); a wavefront owns 32 keys and walks the queries (of its part, where they are split) of all
// the heads that share its key / value head, BLK at a time: their gradients sum in registers.  SUM (LINE): the table's gradient is wanted, its partials go to the slab
template <typename T, int DP, int NW, int BIAS, bool SUM>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP == 128 || sizeof(T) == 4 ? 1 : 2))) void rel_k_kernel(RelP p) {
    constexpr int NT = 64 * NW, BLKN = blk<T>(), KT = BLKN / 32, NCH = DP * (int)sizeof(T) / 32, ND = DP / 32;
    constexpr int IMG = BLKN * DP * (int)sizeof(T), WIN = (32 * NW + BLKN) * 4;
    constexpr int BUF = 2 * IMG + 2 * BLKN * 4 + (BIAS == LINE ? WIN : BIAS == NONE ? 0 : BLKN * 4);
    constexpr bool AHEAD = sizeof(T) == 2 && DP != 64;               // (width 64: two wavefronts a SIMD leave no registers for it)
    extern __shared__ __attribute__((aligned(16))) char lds[];       // [2][Q image | dO image | lse | delta | window or places], BOX: the table
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = lane >> 5;
    const int hk = blockIdx.y, b = blockIdx.z, rep = p.H / p.Hkv;
    const int split = blockIdx.x % p.ksplit, kt0 = blockIdx.x / p.ksplit * NW, k0 = kt0 * 32, key = k0 + wv * 32 + (lane & 31), keyc = min(key, p.Nk - 1);
    const bool kok = key < p.Nk && (!p.mask || p.mask[(long)b * p.Nk + keyc]);
    const int nqb_all = (p.Nq + BLKN - 1) / BLKN, qb0 = (int)((long)split * nqb_all / p.ksplit), nqb = (int)((long)(split + 1) * nqb_all / p.ksplit) - qb0, steps = nqb * rep;
    const int qs0 = qb0 * BLKN;                                          // the part's first query

    u32x4 kf[NCH], vf[NCH];
    {
        const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + (long)b * p.ks[0] + (long)keyc * p.ks[1] + (long)hk * p.ks[2]);
        const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + (long)b * p.vs[0] + (long)keyc * p.vs[1] + (long)hk * p.vs[2]);
#pragma unroll
        for (int s = 0; s < NCH; ++s) {
            kf[s] = vf[s] = (u32x4){0u, 0u, 0u, 0u};
            if (kok && 32 * s + 16 * h < p.D * (int)sizeof(T)) {
                kf[s] = *reinterpret_cast<const u32x4*>(kp + 32 * s + 16 * h);
                vf[s] = *reinterpret_cast<const u32x4*>(vp + 32 * s + 16 * h);
            }
        }
    }
    const int ak = (BIAS == BOX || BIAS == GATHER) ? p.omax - place(p, keyc) : 0;
    float* tab = reinterpret_cast<float*>(lds + 2 * BUF);               // BOX
    // LINE: dS of this wavefront, 32 keys x 32 queries as [key][query], rows of 36 zeros + 32 values (b128 writes of 16 keys cover the banks once; what is read
    // before or behind a row's values is 0)
    constexpr int SK = 68, SKEW = 32 * SK + 36;
    float* skew = reinterpret_cast<float*>(lds + 2 * BUF) + wv * SKEW;
    float run = 0.f;                                                    // running sum of offset (query tile) - (key tile) + lane - 32
    if (SUM)
        for (int i = lane; i < SKEW; i += 64) skew[i] = 0.f;
    const int ktile = kt0 + wv, ktiles = (p.Nk + 31) / 32;
    const bool any = __syncthreads_or(kok);                             // a workgroup whose keys are all masked has only zeros to store

    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) { dk[dt] = zero16(); dv[dt] = zero16(); }

    Tile<T, DP, NT> qt_, dt_;
    float lr = 0.f, tr = 0.f;
    int qpos = 0;
    constexpr int NWIN = (32 * NW + BLKN + NT - 1) / NT;
    float win[BIAS == LINE ? NWIN : 1];
    constexpr bool HALVES = sizeof(T) == 2 && DP == 128;               // as in rel_q_kernel
    auto fetch_d = [&](int it) {
        const int head = hk * rep + it / nqb, q0 = qs0 + (it % nqb) * BLKN, last = min(p.Nq - 1 - q0, BLKN - 1);
        dt_.fetch(static_cast<const T*>(p.dout) + (((long)b * p.Nq + q0) * p.H + head) * p.D, p.H * p.D * (int)sizeof(T), last, p.D, tid);
    };
    auto fetch = [&](int it) {
        const int head = hk * rep + it / nqb, q0 = qs0 + (it % nqb) * BLKN, last = min(p.Nq - 1 - q0, BLKN - 1);
        qt_.fetch(static_cast<const T*>(p.q) + (long)b * p.qs[0] + (long)head * p.qs[2] + q0 * p.qs[1], (int)(p.qs[1] * sizeof(T)), last, p.D, tid);
        if (!HALVES) fetch_d(it);
        if (tid < BLKN) {
            const bool ok = q0 + tid < p.Nq;
            const long lrow = ((long)b * p.H + head) * p.Nq + q0 + tid;
            lr = ok ? p.lse[lrow] : INFINITY;                           // queries past the end: p = 0
            tr = ok ? -p.delta[lrow] : 0.f;
            if (BIAS == BOX || BIAS == GATHER) qpos = place(p, p.q0 + min(q0 + tid, p.Nq - 1));
        }
        if (BIAS == LINE) {
            const int first = p.q0 + q0 - (k0 + 32 * NW - 1) + p.gw - 1;
#pragma unroll
            for (int i = 0; i < NWIN; ++i) {
                const int at = first + i * NT + tid;
                win[i] = (i * NT + tid < 32 * NW + BLKN && at >= 0 && at < p.nd) ? p.e[(long)head * p.nd + at] : 0.f;
            }
        }
    };
    auto commit_q = [&](char* buf, int it) { qt_.commit(buf, tid, first_rows(p.Nq - qs0 - (it % nqb) * BLKN) & Tile<T, DP, NT>::all_rows(), p.D); };
    auto commit = [&](char* buf, int it) {
        if (!HALVES) commit_q(buf, it);
        dt_.commit(buf + IMG, tid, first_rows(p.Nq - qs0 - (it % nqb) * BLKN) & Tile<T, DP, NT>::all_rows(), p.D);
        float* side = reinterpret_cast<float*>(buf + 2 * IMG);
        if (tid < BLKN) {
            side[tid] = lr;
            side[BLKN + tid] = tr;
            if (BIAS == BOX || BIAS == GATHER) reinterpret_cast<int*>(side)[2 * BLKN + tid] = qpos;
        }
        if (BIAS == LINE) {
#pragma unroll
            for (int i = 0; i < NWIN; ++i)
                if (i * NT + tid < 32 * NW + BLKN) side[2 * BLKN + i * NT + tid] = win[i];
        }
    };
    if (SUM && !any && ktile < ktiles)                         // its slab rows are folded all the same
        for (int g = 0; g < rep; ++g) {
            float* row = p.slab + ((((long)b * p.H + hk * rep + g) * ktiles + ktile) * p.ksplit + split) * p.slab_len;
            for (int i = lane; i < p.slab_len; i += 64) row[i] = 0.f;
        }
    auto step = [&](int it, auto between) {
        const int head = hk * rep + it / nqb;
        const char* qimg = lds + (it & 1) * BUF;
        const char* dimg = qimg + IMG;
        const float* lsev = reinterpret_cast<const float*>(qimg + 2 * IMG);
        const float* dltv = lsev + BLKN;
        const float* wl = lsev + 2 * BLKN + (32 * NW - 1 - (wv * 32 + (lane & 31)) + 4 * h);
        f32x16 sa[KT], da[KT];                                           // S and dP - delta of the whole block first: the matrix pipe works on while the vector pipe starts
#pragma unroll
        for (int qt = 0; qt < KT; ++qt) {
            RowFrags<T, DP> qa, oa;
            qa.load(qimg, qt * 32, lane);
            oa.load(dimg, qt * 32, lane);
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(dltv + qt * 32 + 8 * g4 + 4 * h);       // -delta
#pragma unroll
                for (int j = 0; j < 4; ++j) da[qt][4 * g4 + j] = d4[j];
            }
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
            sa[qt] = qa.times(kf, zero16());
            da[qt] = oa.times(vf, da[qt]);
        }
#pragma unroll
        for (int qt = 0; qt < KT; ++qt) {
            TrFrags<T, DP, AHEAD> td, tq;
            td.load(dimg, qt * 32, lane);
            tq.load(qimg, qt * 32, lane);
            // what the 16 scores of a lane need from LDS, requested together (a read at a time would be waited for at a time)
            f32x16 e = zero16(), l = zero16();
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int r0 = qt * 32 + 8 * g4 + 4 * h;
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(lsev + r0);
                int4 qp;
                if (BIAS == BOX || BIAS == GATHER) qp = *reinterpret_cast<const int4*>(lsev + 2 * BLKN + r0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 4 * g4 + j;
                    l[r] = l4[j];
                    if (BIAS == NONE) continue;
                    const int o_ = ak + (j == 0 ? qp.x : j == 1 ? qp.y : j == 2 ? qp.z : qp.w);
                    e[r] = BIAS == LINE ? wl[qt * 32 + 8 * g4 + j] : BIAS == BOX ? tab[o_] : gather_bias(p, head, o_);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = BIAS == NONE ? __builtin_fmaf(sa[qt][r], p.c, -l[r]) : __builtin_fmaf(sa[qt][r], p.c, e[r]) - l[r];
                const float pr = __builtin_amdgcn_exp2f(x);
                sa[qt][r] = pr * da[qt][r];                             // dS
                da[qt][r] = pr;                                         // P   (a lane's columns are its own key's: a masked key's are not stored)
            }
            if (SUM) {
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const f32x4 v = {sa[qt][4 * g4], sa[qt][4 * g4 + 1], sa[qt][4 * g4 + 2], sa[qt][4 * g4 + 3]};
                    *reinterpret_cast<f32x4*>(skew + (lane & 31) * SK + 36 + 8 * g4 + 4 * h) = kok ? v : (f32x4){0.f, 0.f, 0.f, 0.f};
                }
            }
            float diag[SUM ? 32 : 1];
            if (SUM) {
                // along the diagonals: lane l takes query - key = l - 32 of every key kk.  The lower half's offsets end with this tile of queries, the upper half's
                // are the lower half's of the next one
#pragma unroll
                for (int kk = 0; kk < 32; ++kk) diag[kk] = skew[kk * (SK + 1) + 4 + lane];
                __builtin_amdgcn_sched_barrier(0);
            }
            td.product(da[qt], dv, lane);
            tq.product(sa[qt], dk, lane);
            if constexpr (sizeof(T) == 2 && DP == 32) tq.product(rest(sa[qt]), dk, lane);
            if (SUM) {
#pragma unroll
                for (int kk = 0; kk < 32; ++kk) run += diag[kk];
                float* row = p.slab + ((((long)b * p.H + head) * ktiles + min(ktile, ktiles - 1)) * p.ksplit + split) * p.slab_len + (it % nqb) * BLKN + qt * 32;
                const bool end = qt == KT - 1 && (it + 1) % nqb == 0;
                if (ktile < ktiles && (lane < 32 || end)) row[lane] = run;
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(run), 0u, false, false);
                run = end ? 0.f : __uint_as_float(sw[1]);
            }
            if (qt == 0) between();
        }
    };
    auto table_of = [&](int it) {                                          // BOX: the next head's table (the step before ended on a barrier)
        if (BIAS == BOX && it % nqb == 0) {
            const int head = hk * rep + it / nqb;
            for (int i = tid; i < p.nd; i += NT) tab[i] = p.e[(long)head * p.nd + i];
            __syncthreads();
        }
    };
    if (any) {
        fetch(0);
        if (HALVES) { commit_q(lds, 0); fetch_d(0); }
        commit(lds, 0);
        __syncthreads();
        for (int it = 0; it + 1 < steps; ++it) {
            char* next = lds + ((it + 1) & 1) * BUF;
            table_of(it);
            fetch(it + 1);
            step(it, [&] {
                if (HALVES) { commit_q(next, it + 1); fetch_d(it + 1); }
            });
            commit(next, it + 1);
            __syncthreads();
        }
        table_of(steps - 1);
        step(steps - 1, [] {});
    }
    if (key < p.Nk) {
        const long at = (((long)b * p.Nk + key) * p.Hkv + hk) * p.D;
        const float f = p.ksplit > 1 ? 1.f : p.scale;
        const long part = (long)p.B * p.Nk * p.Hkv * p.D;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d = dt * 32 + 8 * g4 + 4 * h;
                if (d >= p.D) continue;
                f32x4 a = {0.f, 0.f, 0.f, 0.f}, c = a;
                if (kok) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) { a[j] = dk[dt][4 * g4 + j] * f; c[j] = dv[dt][4 * g4 + j]; }
                }
                if (p.ksplit > 1) {
                    store4(p.po + split * part + at + d, a);
                    store4(p.po + (p.ksplit + split) * part + at + d, c);
                    continue;
                }
                store4(static_cast<T*>(p.dk) + at + d, a);
                store4(static_cast<T*>(p.dv) + at + d, c);
            }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// dS summed over the batch and over repeated cells, for every pair of cells: M[z][h][a][c], a < QC the queries a, a + QC, ..., c < KC the keys c, c + KC, ....  QC and KC
// are the grid's cells (or all tokens, if they are fewer); of a grid smaller than a tile, as many of its copies as a tile holds.
// grid (query tiles of 32 NW x key blocks, H, parts z of the passes (batch, query copy, key copy)).  Tiles as in rel_q_kernel
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP == 128 || sizeof(T) == 4 ? 1 : 2))) void rel_d_kernel(RelP p) {
    constexpr int NT = 64 * NW, BLKN = blk<T>(), KT = BLKN / 32, NCH = DP * (int)sizeof(T) / 32;
    constexpr int IMG = BLKN * DP * (int)sizeof(T), BUF = 2 * IMG;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = lane >> 5;
    const int nkb = (p.KC + BLKN - 1) / BLKN, head = blockIdx.y, hk = head / (p.H / p.Hkv);
    const int a = ((blockIdx.x / nkb) * NW + wv) * 32 + (lane & 31), c0 = (blockIdx.x % nkb) * BLKN;
    const int MQ = (p.Nq + p.QC - 1) / p.QC, MK = (p.Nk + p.KC - 1) / p.KC;
    const long passes = (long)p.B * MQ * MK;                       // (past 2^31 for long sequences over few cells)
    const long t0 = passes * blockIdx.z / gridDim.z, t1 = passes * (blockIdx.z + 1) / gridDim.z;
    struct Pass { int b, cq, ck; };                                // batch entry, copy of the queries, copy of the keys
    auto next = [&](Pass t) {
        if (++t.ck == MK) { t.ck = 0; if (++t.cq == MQ) { t.cq = 0; ++t.b; } }
        return t;
    };

    f32x16 acc[KT], bias[KT];
    const int aq = place(p, p.q0 + min(a, p.QC - 1)) + p.omax;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        acc[kt] = zero16();
#pragma unroll
        for (int r = 0; r < 16; ++r) bias[kt][r] = p.e[(long)head * p.nd + aq - place(p, min(c0 + kt * 32 + (r & 3) + 8 * (r >> 2) + 4 * h, p.KC - 1))];
    }
    u32x4 qf[NCH], df[NCH];
    float lse2 = INFINITY, dlt = 0.f;
    Tile<T, DP, NT> kt_, vt_;
    uint64_t valid = 0;
    bool there = false;
    auto fetch = [&](Pass t) {
        // (a copy of the cells may end before this block of them does: its rows are then the last token's, and none is valid)
        const int b = t.b, j0 = min(t.ck * p.KC + c0, p.Nk - 1), n = min(p.Nk, (t.ck + 1) * p.KC) - (t.ck * p.KC + c0), last = max(0, min(n, BLKN) - 1);
        kt_.fetch(static_cast<const T*>(p.k) + (long)b * p.ks[0] + (long)hk * p.ks[2] + j0 * p.ks[1], (int)(p.ks[1] * sizeof(T)), last, p.D, tid);
        vt_.fetch(static_cast<const T*>(p.v) + (long)b * p.vs[0] + (long)hk * p.vs[2] + j0 * p.vs[1], (int)(p.vs[1] * sizeof(T)), last, p.D, tid);
        there = lane < min(n, BLKN);
        if (p.mask) there = there && p.mask[(long)b * p.Nk + j0 + min(lane, last)];
    };
    auto commit = [&](char* buf) {
        valid = __ballot(there);
        kt_.commit(buf, tid, valid, p.D);
        vt_.commit(buf + IMG, tid, valid, p.D);
    };
    auto step = [&](Pass t, const char* kimg, bool first) {
        if (first || t.ck == 0) {                                  // the next (batch, query copy)
            const int b = t.b, i = t.cq * p.QC + a, ic = min(i, p.Nq - 1);
            const bool qok = a < p.QC && i < p.Nq;
            const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(p.q) + (long)b * p.qs[0] + (long)ic * p.qs[1] + (long)head * p.qs[2]);
            const char* dp = reinterpret_cast<const char*>(static_cast<const T*>(p.dout) + (((long)b * p.Nq + ic) * p.H + head) * p.D);
#pragma unroll
            for (int s = 0; s < NCH; ++s) {
                const bool in = 32 * s + 16 * h < p.D * (int)sizeof(T);
                const int col = in ? 32 * s + 16 * h : 0;
                const u32x4 u = *reinterpret_cast<const u32x4*>(qp + col), w = *reinterpret_cast<const u32x4*>(dp + col), zero = {0u, 0u, 0u, 0u};
                qf[s] = qok && in ? u : zero;
                df[s] = qok && in ? w : zero;
            }
            const long lrow = ((long)b * p.H + head) * p.Nq + ic;
            lse2 = qok ? p.lse[lrow] : INFINITY;
            dlt = qok ? p.delta[lrow] : 0.f;
        }
        if (valid) {
            const uint64_t vh = h ? valid >> 4 : valid;      // (constant shifts: see row_bit)
            const bool full = valid == Tile<T, DP, NT>::all_rows();
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                RowFrags<T, DP> kf, vf;
                kf.load(kimg, kt * 32, lane);
                vf.load(kimg + IMG, kt * 32, lane);
                __builtin_amdgcn_sched_barrier(0);
                f32x16 st = zero16(), dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] = -dlt;
                st = kf.times(qf, st);
                dp = vf.times(df, dp);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], p.c, bias[kt][r]) - lse2) * dp[r];
                    if (!full) v = (vh >> (kt * 32 + (r & 3) + 8 * (r >> 2))) & 1 ? v : 0.f;
                    acc[kt][r] += v;
                }
            }
        }
    };
    if (t0 < t1) {
        Pass at = {(int)(t0 / MK / MQ), (int)(t0 / MK % MQ), (int)(t0 % MK)};
        fetch(at);
        commit(lds);
        __syncthreads();
        for (long t = t0; t + 1 < t1; ++t) {
            const Pass then = next(at);
            fetch(then);
            step(at, lds + ((t - t0) & 1) * BUF, t == t0);
            commit(lds + ((t + 1 - t0) & 1) * BUF);
            __syncthreads();
            at = then;
        }
        step(at, lds + ((t1 - 1 - t0) & 1) * BUF, t0 + 1 == t1);
    }
    if (a < p.QC) {
        float* dst = p.slab + (((long)blockIdx.z * p.H + head) * p.QC + a) * ((long)nkb * BLKN) + c0 + 4 * h;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                store4(dst + kt * 32 + 8 * g4, (f32x4){acc[kt][4 * g4], acc[kt][4 * g4 + 1], acc[kt][4 * g4 + 2], acc[kt][4 * g4 + 3]});
    }
}

template <typename K> int grant_lds(K kern, int bytes) {
    if (bytes > 64 * 1024) HIP_RET(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return 0;
}

template <typename T, int DP, int NW, int MODE, int BIAS>
int launch_q(const RelP& p, hipStream_t st) {
    constexpr int BLKN = blk<T>();
    int bytes = 2 * (2 * BLKN * DP * (int)sizeof(T) + (BIAS == LINE ? (p.few ? (p.pack ? p.H / p.Hkv : 1) * (BLKN + p.Nq) * 4 + 15 & ~15 : (32 * NW + BLKN) * 4) : BIAS == NONE ? 0 : BLKN * 4));
    if (BIAS == BOX) bytes += p.nd * 4;
    const int rc = grant_lds(rel_q_kernel<T, DP, NW, MODE, BIAS>, bytes);
    if (rc) return rc;
    const int rows = p.pack ? p.Nq * (p.H / p.Hkv) : p.Nq;
    hipLaunchKernelGGL((rel_q_kernel<T, DP, NW, MODE, BIAS>), dim3((rows + 32 * NW - 1) / (32 * NW) * p.nsplit, p.pack ? p.Hkv : p.H, p.B), dim3(64 * NW), bytes, st, p);
    LAUNCH_RET();
    return 0;
}
template <typename T, int DP, int NW, int BIAS, bool SUM>
int launch_k(const RelP& p, hipStream_t st) {
    constexpr int BLKN = blk<T>();
    int bytes = 2 * (2 * BLKN * DP * (int)sizeof(T) + 2 * BLKN * 4 + (BIAS == LINE ? (32 * NW + BLKN) * 4 : BIAS == NONE ? 0 : BLKN * 4));
    if (BIAS == BOX) bytes += p.nd * 4;
    if (SUM) bytes += NW * (32 * 68 + 36) * 4;
    const int rc = grant_lds(rel_k_kernel<T, DP, NW, BIAS, SUM>, bytes);
    if (rc) return rc;
    hipLaunchKernelGGL((rel_k_kernel<T, DP, NW, BIAS, SUM>), dim3((p.Nk + 32 * NW - 1) / (32 * NW) * p.ksplit, p.Hkv, p.B), dim3(64 * NW), bytes, st, p);
    LAUNCH_RET();
    return 0;
}

template <typename T, int DP, int NW>
int launch_d(const RelP& p, hipStream_t st) {
    constexpr int BLKN = blk<T>(), bytes = 4 * BLKN * DP * (int)sizeof(T);
    const int rc = grant_lds(rel_d_kernel<T, DP, NW>, bytes);
    if (rc) return rc;
    hipLaunchKernelGGL((rel_d_kernel<T, DP, NW>), dim3((p.QC + 32 * NW - 1) / (32 * NW) * ((p.KC + BLKN - 1) / BLKN), p.H, p.parts), dim3(64 * NW), bytes, st, p);
    LAUNCH_RET();
    return 0;
}

template <typename T, int DP, int NW>
int pick_bias(const RelP& p, int what, hipStream_t st) {
    if (what == 3) return launch_d<T, DP, NW>(p, st);
    if (what == 2 && p.bias == LINE && p.slab) return launch_k<T, DP, NW, LINE, true>(p, st);
#define REL_ONE(BIAS) (what == 0 ? launch_q<T, DP, NW, 0, BIAS>(p, st) : what == 1 ? launch_q<T, DP, NW, 1, BIAS>(p, st) : launch_k<T, DP, NW, BIAS, false>(p, st))
    switch (p.bias) {
        case NONE: return REL_ONE(NONE);
        case BOX: return REL_ONE(BOX);
        case LINE: return REL_ONE(LINE);
        default: return REL_ONE(GATHER);
    }
#undef REL_ONE
}
template <typename T, int DP>
int pick_nw(const RelP& p, int what, int nw, hipStream_t st) {
    return nw == 4 ? pick_bias<T, DP, 4>(p, what, st) : nw == 2 ? pick_bias<T, DP, 2>(p, what, st) : pick_bias<T, DP, 1>(p, what, st);
}

}  // namespace
