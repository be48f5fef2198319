// What a training block does around its recurrence and products, each in one
// pass over the rows (RWKVBlock.swift:163-307, which the reference forms from
// MLX operations): dropout from a counter-based generator, the join of one
// block with the next (norm, gate, dropout and scale of the branch, the
// residual sum, the next norm), and the recurrence's tail (head norm, bonus,
// gate) with its gradients.
//
//   dropout   y = res + m·x,  dx = m·dy
//   join      n = LN(o; w1, b1), x' = x + s·m·(g·n), h = LN(x'; w, b)
//   tail      y = (LN64(o)·w + b + (Σ_head r·k·r_k)·v)·g
//
// m of row r, columns 8c .. 8c + 7: the 128 bits of Philox4x32-10 (Salmon,
// Moraes, Dror, Shaw 2011) for the key `seed` and the counter (c, r, offset)
// are eight 16-bit numbers; a value whose number is under t = round(65536·p)
// is dropped, the others are multiplied by 65536/(65536 − t).  No mask is
// stored: the backward pass draws the numbers again.  16 bits a value, not 32,
// halve the generator's work, 20 products of 32 x 32 bits a draw.
//
// Statistics, sums and gradients are fp32; one rounding per output.  Column
// sums: a block's rows in registers, one partial row per block, joined in a
// fixed order (no atomics: the same bits every time).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "act8.h"
#include "launch.h"
#include "wkv7_step.h"

namespace {

using namespace rwkv_train;
typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int JOIN_MAX_D = 8192;   // 1024 threads of a chunk each
constexpr int HEAD = 64;

// ───────────────────────────── random numbers ─────────────────────────────

struct Drop {
    uint64_t seed;
    const int64_t* seed_dev;   // the seed, where not null
    uint64_t offset;
    uint32_t threshold;        // 0: everything is kept
    float scale;
    __device__ __forceinline__ uint64_t key() const { return seed_dev ? (uint64_t)*seed_dev : seed; }
};

// The eight 16-bit numbers of chunk c of a row, two a word.
__device__ __forceinline__ uint4 numbers(uint32_t c, uint32_t row, uint64_t offset, uint64_t key) {
    uint32_t c0 = c, c1 = row, c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// m of the eight values, as what they are multiplied by; a dropped value has 0.
__device__ __forceinline__ void factors(const Drop& d, uint64_t key, uint32_t c, uint32_t row, float (&m)[8]) {
    const uint4 q = numbers(c, row, d.offset, key);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = (i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu) >= d.threshold ? d.scale : 0.0f;
}

// A dropped value is zero whatever it was, an infinity or a NaN too.
__device__ __forceinline__ float dropped(float m, float v) { return m > 0.0f ? m * v : 0.0f; }

// ───────────────────────────── dropout ─────────────────────────────

struct DropoutArgs {
    const void* x;
    int64_t ldx;
    const void* res;   // of y's type, or null
    int64_t ldr;
    void* y;           // [N, D]
    int64_t chunks;    // N·cpr
    int cpr, D;        // chunks of 8 a row
    uint32_t magic;    // ceil(2^32 / cpr) where cpr is at most a block's chunks
    Drop drop;
};

// Chunks of 8 values, U a thread, a block's in one run; its first row is found
// once (in 64 bits), the others from there: a quotient under 2·RUN by a divisor
// of at most RUN is the high half of a 32-bit product with ceil(2^32 / cpr).
constexpr int DROP_U = 4, DROP_RUN = 256 * DROP_U;

template <typename TX, typename TY>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const int64_t first = (int64_t)blockIdx.x * DROP_RUN;
    const int64_t row0 = first / a.cpr;
    const uint32_t rem = (uint32_t)(first - row0 * a.cpr);
    const int left = (int)min(a.chunks - first, (int64_t)DROP_RUN);
    const uint64_t key = a.drop.key();
    Raw8<TX> x[DROP_U];
    Raw8<TY> r[DROP_U];
    int64_t row[DROP_U];
    uint32_t c[DROP_U];
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
        const int at = threadIdx.x + 256 * u;
        const uint32_t n = rem + at;
        const uint32_t q = a.cpr == 1 ? n : a.cpr > DROP_RUN ? (n >= (uint32_t)a.cpr) : __umulhi(n, a.magic);
        row[u] = row0 + q;
        c[u] = n - q * a.cpr;
        if (at >= left) continue;
        x[u].load(reinterpret_cast<const TX*>(a.x) + row[u] * a.ldx + 8 * c[u], a.D - 8 * (int)c[u]);
        if (a.res) r[u].load(reinterpret_cast<const TY*>(a.res) + row[u] * a.ldr + 8 * c[u], a.D - 8 * (int)c[u]);
    }
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
        if ((int)threadIdx.x + 256 * u >= left) continue;
        float v[8], m[8];
        x[u].get(v);
        if (a.drop.threshold) {
            factors(a.drop, key, c[u], (uint32_t)row[u], m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = dropped(m[i], v[i]);
        }
        if (a.res) {
            r[u].get(m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += m[i];
        }
        store8(reinterpret_cast<TY*>(a.y) + row[u] * a.D + 8 * c[u], a.D - 8 * (int)c[u], v);
    }
}

// ───────────────────────────── join ─────────────────────────────

// Sums of two values over the TPR threads of a row, as row_sum of the layer
// norm takes one: one wave, or the block through LDS, the waves in order.
// Every thread has read a slot before the barrier of the next sum, so two
// slots in turn are enough.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float s, float q, float2 (*part)[16], int slot) {
    s = rwkv_wkv::wave_total(s);
    q = rwkv_wkv::wave_total(q);
    if constexpr (TPR == 64) {
        return make_float2(s, q);
    } else {
        if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = make_float2(s, q);
        __syncthreads();
        float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) t.x += part[slot][i].x, t.y += part[slot][i].y;
        return t;
    }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float2 (*part)[16], int slot) {
    s = rwkv_wkv::wave_total(s);
    if constexpr (TPR == 64) {
        return s;
    } else {
        if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6].x = s;
        __syncthreads();
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) t += part[slot][i].x;
        return t;
    }
}

template <typename T>
__device__ __forceinline__ void load_w(const void* w, int w32, int col, int valid, float (&v)[8]) {
    if (w32)
        load8(reinterpret_cast<const float*>(w) + col, valid, v);
    else
        load8(reinterpret_cast<const T*>(w) + col, valid, v);
}

struct JoinFwd {
    const void *x, *o, *gate;   // gate, post_w, post_b, scale, b may be null
    int64_t ldx, ldo, ldg;
    const void *post_w, *post_b, *scale, *w, *b;
    int w32;                    // the vectors are fp32 (else o's type)
    void *xs, *h;               // [N, D]
    float* stats;               // [N, 4]: mean and rstd of o, of x'; or null
    int64_t N;
    int D;
    float post_eps, eps;
    Drop drop;
};

// Rows blockIdx.x·RPB + threadIdx.x / TPR, + gridDim.x·RPB, ...; a thread holds
// one chunk of 8 columns of a row and the vectors' values for it.
template <typename TS, typename T, int TPR>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void join_fwd_kernel(JoinFwd a) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float2 part[2][16];
    const int t = threadIdx.x % TPR, col = 8 * t, valid = a.D - col;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= a.N) return;   // whole waves; rows that share a barrier end together
    const float n = (float)a.D;
    const uint64_t key = a.drop.threshold ? a.drop.key() : 0;
    float pw[8], pb[8], sc[8], w[8], b[8];
    if (a.post_w) load_w<T>(a.post_w, a.w32, col, valid, pw);
    if (a.post_b) load_w<T>(a.post_b, a.w32, col, valid, pb);
    if (a.scale) load_w<T>(a.scale, a.w32, col, valid, sc);
    load_w<T>(a.w, a.w32, col, valid, w);
    if (a.b) load_w<T>(a.b, a.w32, col, valid, b);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = 0.0f;
    for (; row < a.N; row += step) {
        float v[8], u[8], g[8];
        load8(reinterpret_cast<const T*>(a.o) + row * a.ldo + col, valid, u);
        load8(reinterpret_cast<const TS*>(a.x) + row * a.ldx + col, valid, v);
        if (a.gate) load8(reinterpret_cast<const T*>(a.gate) + row * a.ldg + col, valid, g);
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.post_w) {
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += u[i];
            st.x = row_sum<TPR>(s, part, 0) / n;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = u[i] - st.x;
                q += col + i < a.D ? d * d : 0.0f;
            }
            st.y = 1.0f / sqrtf(row_sum<TPR>(q, part, 1) / n + a.post_eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = (u[i] - st.x) * st.y * pw[i];
            if (a.post_b)
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] += pb[i];
        }
        if (a.gate)
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= g[i];
        if (a.drop.threshold) {
            factors(a.drop, key, (uint32_t)t, (uint32_t)row, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = dropped(g[i], u[i]);
        }
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = col + i < a.D ? v[i] + (a.scale ? sc[i] * u[i] : u[i]) : 0.0f;
            s += v[i];
        }
        if (valid > 0) store8(reinterpret_cast<TS*>(a.xs) + row * a.D + col, valid, v);
        st.z = row_sum<TPR>(s, part, 0) / n;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = v[i] - st.z;
            q += col + i < a.D ? d * d : 0.0f;
        }
        st.w = 1.0f / sqrtf(row_sum<TPR>(q, part, 1) / n + a.eps);
        if (a.stats && t == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = st;
        if (valid <= 0) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (v[i] - st.z) * st.w * w[i] + b[i];
        store8(reinterpret_cast<T*>(a.h) + row * a.D + col, valid, v);
    }
}

enum { DW, DB, DPW, DPB, DSC, SUMS };   // column sums of the join

struct JoinBwd {
    const void *xs, *o, *gate;  // o null: it does not reach a gradient
    int64_t ldo, ldg;
    const float* stats;
    const void *post_w, *post_b, *scale, *w;
    int w32;
    const void *dxs, *dh;       // [N, D], either may be null: zeros
    void *dx, *dout, *dgate;    // [N, D], each may be null
    float* part;                // [gridDim.x][sums][D]
    int slot[SUMS];             // a sum's place, or -1
    int sums;
    int64_t N;
    int D;
    Drop drop;
};

// With xh = (x' − μ)·r and G the whole gradient of x':
//   G = dx' + LN'(dh·w; xh, r), dw = Σ dh·xh, db = Σ dh
//   du = G·s·m, ds = Σ G·m·u, dg = du·n, dn = du·g
//   do = LN'(dn·w1; oh, r1), dw1 = Σ dn·oh, db1 = Σ dn
// LN'(y; h, r) = r·(y − mean y − h·mean(y·h)).
template <typename TS, typename T, int TPR>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void join_bwd_kernel(JoinBwd a) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float2 part[2][16];
    __shared__ float sums[RPB > 1 ? 4 * 8 * 64 : 1];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, col = 8 * t, valid = a.D - col;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float n = (float)a.D;
    const uint64_t key = a.drop.threshold ? a.drop.key() : 0;
    float pw[8], pb[8], sc[8], w[8];
    auto vectors = [&] {
        if (a.post_w) load_w<T>(a.post_w, a.w32, col, valid, pw);
        if (a.post_b) load_w<T>(a.post_b, a.w32, col, valid, pb);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) pb[i] = 0.0f;
        if (a.scale) load_w<T>(a.scale, a.w32, col, valid, sc);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i] = 1.0f;
        load_w<T>(a.w, a.w32, col, valid, w);
    };
    if constexpr (TPR < 1024) vectors();   // 1024 threads have 128 registers each: read row by row
    float acc[SUMS][8] = {};
    int slot = 0;
    for (int64_t row = (int64_t)blockIdx.x * RPB + grp; row < a.N; row += step) {
        float G[8], y[8], xh[8], u[8], g[8];
        const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * row);
        if constexpr (TPR == 1024) vectors();
        if (a.dxs) load8(reinterpret_cast<const TS*>(a.dxs) + row * a.D + col, valid, G);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) G[i] = 0.0f;
        if (a.o) load8(reinterpret_cast<const T*>(a.o) + row * a.ldo + col, valid, u);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = 0.0f;
        if (a.gate) load8(reinterpret_cast<const T*>(a.gate) + row * a.ldg + col, valid, g);
        if (a.dh) {
            load8(reinterpret_cast<const T*>(a.dh) + row * a.D + col, valid, y);
            load8(reinterpret_cast<const TS*>(a.xs) + row * a.D + col, valid, xh);
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                xh[i] = i < valid ? (xh[i] - st.z) * st.w : 0.0f;
                acc[DW][i] += y[i] * xh[i];
                acc[DB][i] += y[i];
                y[i] *= w[i];
                s1 += y[i];
                s2 += y[i] * xh[i];
            }
            const float2 s = row_sum2<TPR>(s1, s2, part, slot);
            slot ^= 1;
            s1 = s.x / n, s2 = s.y / n;
#pragma unroll
            for (int i = 0; i < 8; ++i) G[i] += (y[i] - s1 - xh[i] * s2) * st.w;
        }
        if (a.dx && valid > 0) store8(reinterpret_cast<TS*>(a.dx) + row * a.D + col, valid, G);
        float m[8], oh[8];
        if (a.drop.threshold) factors(a.drop, key, (uint32_t)t, (uint32_t)row, m);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i] = 1.0f;
        float p1 = 0.0f, p2 = 0.0f;
        // u: n, then dn·w1; y: dg
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            oh[i] = a.post_w ? (i < valid ? (u[i] - st.x) * st.y : 0.0f) : u[i];
            const float nv = a.post_w ? oh[i] * pw[i] + pb[i] : u[i], gv = a.gate ? g[i] : 1.0f;
            const float gm = dropped(m[i], i < valid ? G[i] : 0.0f);   // past the row's end G is not zero
            acc[DSC][i] += m[i] > 0.0f ? gm * (gv * nv) : 0.0f;
            const float du = gm * sc[i];
            y[i] = du * nv;
            const float dn = du * gv;
            acc[DPW][i] += dn * oh[i];
            acc[DPB][i] += dn;
            u[i] = a.post_w ? dn * pw[i] : dn;
            p1 += u[i];
            p2 += u[i] * oh[i];
        }
        if (a.dgate && valid > 0) store8(reinterpret_cast<T*>(a.dgate) + row * a.D + col, valid, y);
        if (!a.dout) continue;
        if (a.post_w) {
            const float2 p = row_sum2<TPR>(p1, p2, part, slot);
            slot ^= 1;
            p1 = p.x / n, p2 = p.y / n;
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = (u[i] - p1 - oh[i] * p2) * st.y;
        }
        if (valid > 0) store8(reinterpret_cast<T*>(a.dout) + row * a.D + col, valid, u);
    }
    if (!a.part) return;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        if (a.slot[k] < 0) continue;   // the same for all
        if constexpr (RPB > 1) {
            // the block's row groups meet in order
            __syncthreads();
            if (grp > 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[(grp * 8 + i) * 64 + t] = acc[k][i];
            __syncthreads();
            if (grp == 0)
#pragma unroll
                for (int r = 1; r < RPB; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[k][i] += sums[(r * 8 + i) * 64 + t];
        }
        if (grp == 0 && valid > 0)
            store8(a.part + ((int64_t)blockIdx.x * a.sums + a.slot[k]) * a.D + col, valid, acc[k]);
    }
}

struct Outs {
    void* p[SUMS];
};

// Column sums of part [G][sums][D] (G may be 0) into out.p[0 .. sums): a block
// owns 16 columns of one sum and splits the G rows over 16 thread rows, each in
// order; the 16 partial sums meet in LDS, in order.
template <typename T>
__global__ __launch_bounds__(256) void join_reduce_kernel(const float* part, int G, int sums, int D, Outs out) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + c, k = blockIdx.y;
    float t = 0.0f;
    if (col < D) {
#pragma unroll 8
        for (int g = r; g < G; g += 16) t += part[((int64_t)g * sums + k) * D + col];
    }
    s[r][c] = t;
    __syncthreads();
    if (r != 0 || col >= D) return;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += s[i][c];
    T* o = reinterpret_cast<T*>(out.p[0]);
#pragma unroll
    for (int i = 1; i < SUMS; ++i)
        if (k == i) o = reinterpret_cast<T*>(out.p[i]);
    o[col] = (T)sum;
}

// ───────────────────────────── tail ─────────────────────────────

// Sum over eight neighbouring lanes, in all of them: lanes 1 and 2 apart within
// a quad, then the half row mirrored.
__device__ __forceinline__ float sum8(float x) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, false));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, false));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xf, 0xf, false));
    return x;
}

struct TailArgs {
    const void *o, *r, *k, *v, *g;
    int64_t ldo, ldr, ldk, ldv, ldg;
    const void *rk, *w, *b;
    int w32;
    void* y;                              // forward: [N, C]
    const void* dy;                       // backward
    int64_t lddy;
    void *dout, *dr, *dk, *dv, *dg;       // [N, C], each may be null
    float* part;                          // [gridDim.y][3][C]: r_k, w, b; or null
    int64_t N;
    int C;
    float eps;
};

// A head is eight neighbouring lanes of 8 columns; TX lanes across, 256 / TX
// rows down a block, rows strided over gridDim.y.
template <typename TO, typename T>
__global__ __launch_bounds__(256) void tail_fwd_kernel(TailArgs a, int TX) {
    const int tx = threadIdx.x % TX, col = 8 * (blockIdx.x * TX + tx);
    if (col >= a.C) return;   // whole heads
    const int64_t step = (int64_t)gridDim.y * (256 / TX);
    float rk[8], w[8], b[8];
    load_w<T>(a.rk, a.w32, col, 8, rk);
    load_w<T>(a.w, a.w32, col, 8, w);
    load_w<T>(a.b, a.w32, col, 8, b);
    for (int64_t row = (int64_t)blockIdx.y * (256 / TX) + threadIdx.x / TX; row < a.N; row += step) {
        float o[8], r[8], k[8], v[8], g[8];
        load8(reinterpret_cast<const TO*>(a.o) + row * a.ldo + col, 8, o);
        load8(reinterpret_cast<const T*>(a.r) + row * a.ldr + col, 8, r);
        load8(reinterpret_cast<const T*>(a.k) + row * a.ldk + col, 8, k);
        load8(reinterpret_cast<const T*>(a.v) + row * a.ldv + col, 8, v);
        load8(reinterpret_cast<const T*>(a.g) + row * a.ldg + col, 8, g);
        float s = 0.0f, q = 0.0f, d = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s += o[i];
            d += r[i] * k[i] * rk[i];
        }
        const float mean = sum8(s) * (1.0f / HEAD);
        d = sum8(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[i] -= mean;
            q += o[i] * o[i];
        }
        const float inv = 1.0f / sqrtf(sum8(q) * (1.0f / HEAD) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (o[i] * inv * w[i] + b[i] + d * v[i]) * g[i];
        store8(reinterpret_cast<T*>(a.y) + row * a.C + col, 8, o);
    }
}

// With oh = (o − μ)·i, d = Σ r·k·r_k, q = oh·w + b + d·v:
//   dg = dy·q, dq = dy·g, dv = dq·d, e = Σ dq·v, dr = e·k·r_k, dk = e·r·r_k
//   do = LN'(dq·w; oh, i);  dr_k = Σ e·r·k, dw = Σ dq·oh, db = Σ dq
template <typename TO, typename T>
__global__ __launch_bounds__(256) void tail_bwd_kernel(TailArgs a, int TX) {
    __shared__ float sums[8 * 256];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, TY = 256 / TX, col = 8 * (blockIdx.x * TX + tx);
    const bool in = col < a.C;   // whole heads
    const int64_t step = (int64_t)gridDim.y * TY;
    float acc[3][8] = {};
    if (in) {
        float rk[8], w[8], b[8];
        load_w<T>(a.rk, a.w32, col, 8, rk);
        load_w<T>(a.w, a.w32, col, 8, w);
        load_w<T>(a.b, a.w32, col, 8, b);
        for (int64_t row = (int64_t)blockIdx.y * TY + ty; row < a.N; row += step) {
            float o[8], r[8], k[8], v[8], g[8], y[8];
            load8(reinterpret_cast<const TO*>(a.o) + row * a.ldo + col, 8, o);
            load8(reinterpret_cast<const T*>(a.r) + row * a.ldr + col, 8, r);
            load8(reinterpret_cast<const T*>(a.k) + row * a.ldk + col, 8, k);
            load8(reinterpret_cast<const T*>(a.v) + row * a.ldv + col, 8, v);
            load8(reinterpret_cast<const T*>(a.g) + row * a.ldg + col, 8, g);
            load8(reinterpret_cast<const T*>(a.dy) + row * a.lddy + col, 8, y);
            float s = 0.0f, q = 0.0f, d = 0.0f, e = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s += o[i];
                d += r[i] * k[i] * rk[i];
                e += y[i] * g[i] * v[i];
            }
            const float mean = sum8(s) * (1.0f / HEAD);
            d = sum8(d);
            e = sum8(e);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] -= mean;
                q += o[i] * o[i];
            }
            const float inv = 1.0f / sqrtf(sum8(q) * (1.0f / HEAD) + a.eps);
            float m1 = 0.0f, m2 = 0.0f, t[8];
            const int64_t at = row * a.C + col;
            // o: oh; g: dq; t: dg
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] *= inv;
                t[i] = y[i] * (o[i] * w[i] + b[i] + d * v[i]);
                g[i] *= y[i];
                acc[0][i] += e * (r[i] * k[i]);
                acc[1][i] += g[i] * o[i];
                acc[2][i] += g[i];
                m1 += g[i] * w[i];
                m2 += g[i] * w[i] * o[i];
            }
            if (a.dg) store8(reinterpret_cast<T*>(a.dg) + at, 8, t);
            m1 = sum8(m1) * (1.0f / HEAD);
            m2 = sum8(m2) * (1.0f / HEAD);
            if (a.dv) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = g[i] * d;
                store8(reinterpret_cast<T*>(a.dv) + at, 8, t);
            }
            if (a.dr) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = e * (k[i] * rk[i]);
                store8(reinterpret_cast<T*>(a.dr) + at, 8, t);
            }
            if (a.dk) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = e * (r[i] * rk[i]);
                store8(reinterpret_cast<T*>(a.dk) + at, 8, t);
            }
            if (a.dout) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = (g[i] * w[i] - m1 - o[i] * m2) * inv;
                store8(reinterpret_cast<TO*>(a.dout) + at, 8, t);
            }
        }
    }
    if (!a.part) return;
    for (int k = 0; k < 3; ++k) {   // the block's rows of threads meet in order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i * 256 + threadIdx.x] = k == 0 ? acc[0][i] : k == 1 ? acc[1][i] : acc[2][i];
        __syncthreads();
        if (ty != 0 || !in) continue;
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = sums[i * 256 + tx];
        for (int r = 1; r < TY; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += sums[i * 256 + r * TX + tx];
        store8(a.part + ((int64_t)blockIdx.y * 3 + k) * a.C + col, 8, s);
    }
}

// ───────────────────────────── launches ─────────────────────────────

rwkv_status status_of(const char* what) {
    const hipError_t e = hipGetLastError();
    RWKV_REQUIRE(e == hipSuccess, RWKV_E_HIP, "%s: %s", what, hipGetErrorString(e));
    return RWKV_OK;
}

Drop drop_of(const rwkv_drop& d) {
    return Drop{d.seed, d.seed_dev, d.offset, (uint32_t)d.threshold,
                d.threshold < 65536 ? (float)(65536.0 / (65536 - d.threshold)) : 0.0f};
}
bool drop_ok(const rwkv_drop* d) { return d && d->threshold >= 0 && d->threshold <= 65536; }

// One type for both, or one of them fp32.
bool pair_ok(int x, int y) { return rwkv::dtype_ok(x) && rwkv::dtype_ok(y) && (x == y || x == RWKV_F32 || y == RWKV_F32); }

// Runs f with values of the types of (wide, dt), wide being dt or fp32.
template <typename F>
void by_types(int wide, int dt, F f) {
    if (dt == RWKV_BF16) {
        if (wide == RWKV_F32) f(float{}, bf16{});
        else f(bf16{}, bf16{});
    } else if (dt == RWKV_F16) {
        if (wide == RWKV_F32) f(float{}, f16{});
        else f(f16{}, f16{});
    } else {
        f(float{}, float{});
    }
}

template <typename F>
void by_width(int64_t D, F f) {
    if (D <= 512) f(std::integral_constant<int, 64>{});
    else if (D <= 1024) f(std::integral_constant<int, 128>{});
    else if (D <= 2048) f(std::integral_constant<int, 256>{});
    else if (D <= 4096) f(std::integral_constant<int, 512>{});
    else f(std::integral_constant<int, 1024>{});
}

// Blocks of the join's passes: rows beyond a full chip's are walked.
int join_fwd_blocks(int64_t N, int64_t D) {
    const int full = D <= 512 ? 2048 : D <= 1024 ? 4096 : D <= 2048 ? 2048 : D <= 4096 ? 1024 : 512;
    return (int)std::min<int64_t>(D <= 512 ? (N + 3) / 4 : N, full);
}
// Each block writes one partial row per column sum.
int join_bwd_blocks(int64_t N, int64_t D) {
    const int full = D <= 512 ? 768 : D <= 1024 ? 1536 : D <= 2048 ? 768 : D <= 4096 ? 512 : 256;
    return (int)std::min<int64_t>(D <= 512 ? (N + 3) / 4 : N, full);
}

// Lanes across and the grid of the tail's passes.
void tail_geometry(int64_t N, int64_t C, int most, int& TX, int& gx, int& gy) {
    const int64_t chunks = C / 8;
    TX = 8;
    while (TX < 64 && TX < chunks) TX *= 2;
    gx = (int)((chunks + TX - 1) / TX);
    const int ty = 256 / TX;
    gy = (int)std::max<int64_t>(1, std::min<int64_t>((N + ty - 1) / ty, std::max(1, most / gx)));
}
constexpr int TAIL_FWD_BLOCKS = 4096, TAIL_BWD_BLOCKS = 1024;

bool join_ok(const rwkv_join* a) {
    return (a->x_dt == a->dt || a->x_dt == RWKV_F32) && rwkv::dtype_ok(a->dt) && (a->w_dt == RWKV_F32 || a->w_dt == a->dt);
}

}  // namespace

extern "C" {

rwkv_status rwkv_dropout(const void* x, rwkv_dtype x_dt, int64_t ldx, const void* residual, int64_t ldr, void* y,
                         rwkv_dtype y_dt, const rwkv_drop* drop, int64_t N, int64_t D, void* stream) {
    RWKV_REQUIRE(pair_ok(x_dt, y_dt), RWKV_E_DTYPE, "dropout: types x %d, y %d", (int)x_dt, (int)y_dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= (1 << 22) && ldx >= D && (!residual || ldr >= D), RWKV_E_SHAPE,
                 "dropout: N=%lld D=%lld ldx=%lld ldr=%lld", (long long)N, (long long)D, (long long)ldx, (long long)ldr);
    RWKV_REQUIRE(N == 0 || (x && y), RWKV_E_NULL, "dropout: null buffer");
    RWKV_REQUIRE(drop_ok(drop), RWKV_E_UNSUPPORTED, "dropout: threshold %d of 65536", drop ? drop->threshold : -1);
    if (N == 0) return RWKV_OK;
    const int64_t cpr = (D + 7) / 8, chunks = N * cpr, blocks = (chunks + DROP_RUN - 1) / DROP_RUN;
    RWKV_REQUIRE(blocks < (int64_t(1) << 31), RWKV_E_SHAPE, "dropout: %lld values", (long long)(N * D));
    const DropoutArgs a{x, ldx, residual, ldr, y, chunks, (int)cpr, (int)D,
                        (uint32_t)(((uint64_t(1) << 32) + cpr - 1) / cpr), drop_of(*drop)};
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks);
    if (y_dt == RWKV_F32 || x_dt == y_dt) {
        by_types(y_dt, x_dt, [&](auto ty, auto tx) {
            rwkv::launch(dropout_kernel<decltype(tx), decltype(ty)>, grid, dim3(256), s, a);
        });
    } else {
        by_types(x_dt, y_dt, [&](auto tx, auto ty) {
            rwkv::launch(dropout_kernel<decltype(tx), decltype(ty)>, grid, dim3(256), s, a);
        });
    }
    return status_of("dropout launch");
}

rwkv_status rwkv_join_fwd(const rwkv_join* j, void* xs, void* h, float* stats, void* stream) {
    RWKV_REQUIRE(j, RWKV_E_NULL, "join_fwd: null arguments");
    RWKV_REQUIRE(join_ok(j), RWKV_E_DTYPE, "join_fwd: types x %d, o %d, vectors %d", (int)j->x_dt, (int)j->dt, (int)j->w_dt);
    RWKV_REQUIRE(j->N >= 0 && j->N <= (1 << 24) && j->D >= 1 && j->D <= JOIN_MAX_D && j->ldx >= j->D && j->ldo >= j->D &&
                     (!j->gate || j->ldg >= j->D),
                 RWKV_E_SHAPE, "join_fwd: N=%lld D=%lld ldx=%lld ldo=%lld ldg=%lld (D <= %d)", (long long)j->N,
                 (long long)j->D, (long long)j->ldx, (long long)j->ldo, (long long)j->ldg, JOIN_MAX_D);
    RWKV_REQUIRE(j->N == 0 || (j->x && j->o && j->weight && xs && h), RWKV_E_NULL, "join_fwd: null buffer");
    RWKV_REQUIRE(j->post_weight || !j->post_bias, RWKV_E_NULL, "join_fwd: post_bias without post_weight");
    RWKV_REQUIRE((uintptr_t)stats % 16 == 0, RWKV_E_SHAPE, "join_fwd: misaligned stats");
    RWKV_REQUIRE(drop_ok(&j->drop), RWKV_E_UNSUPPORTED, "join_fwd: threshold %d of 65536", j->drop.threshold);
    if (j->N == 0) return RWKV_OK;
    const JoinFwd a{j->x, j->o, j->gate, j->ldx, j->ldo, j->ldg, j->post_weight, j->post_bias, j->scale, j->weight, j->bias,
                    j->w_dt == RWKV_F32, xs, h, stats, j->N, (int)j->D, j->post_eps, j->eps, drop_of(j->drop)};
    const dim3 grid((unsigned)join_fwd_blocks(j->N, j->D));
    by_types(j->x_dt, j->dt, [&](auto ts, auto t) {
        by_width(j->D, [&](auto tpr) {
            constexpr int TPR = decltype(tpr)::value;
            rwkv::launch(join_fwd_kernel<decltype(ts), decltype(t), TPR>, grid, dim3(TPR == 64 ? 256 : TPR),
                         (hipStream_t)stream, a);
        });
    });
    return status_of("join_fwd launch");
}

int64_t rwkv_join_bwd_workspace(int64_t N, int64_t D) {
    if (N < 0 || D < 1 || D > JOIN_MAX_D) return 0;
    return (int64_t)join_bwd_blocks(N, D) * SUMS * D * 4;
}

rwkv_status rwkv_join_bwd(const rwkv_join* j, const void* xs, const float* stats, const void* dxs, const void* dh, void* dx,
                          void* dout, void* dgate, void* dweight, void* dbias, void* dpost_weight, void* dpost_bias,
                          void* dscale, void* workspace, int64_t workspace_bytes, void* stream) {
    RWKV_REQUIRE(j, RWKV_E_NULL, "join_bwd: null arguments");
    RWKV_REQUIRE(join_ok(j), RWKV_E_DTYPE, "join_bwd: types x %d, o %d, vectors %d", (int)j->x_dt, (int)j->dt, (int)j->w_dt);
    RWKV_REQUIRE(j->N >= 0 && j->N <= (1 << 24) && j->D >= 1 && j->D <= JOIN_MAX_D && (!j->o || j->ldo >= j->D) &&
                     (!j->gate || j->ldg >= j->D),
                 RWKV_E_SHAPE, "join_bwd: N=%lld D=%lld ldo=%lld ldg=%lld (D <= %d)", (long long)j->N, (long long)j->D,
                 (long long)j->ldo, (long long)j->ldg, JOIN_MAX_D);
    RWKV_REQUIRE(j->N == 0 || ((j->o || !(j->gate || j->post_weight || j->scale)) && j->weight && xs && stats), RWKV_E_NULL,
                 "join_bwd: null buffer");
    RWKV_REQUIRE((j->post_weight || (!j->post_bias && !dpost_weight && !dpost_bias)) && (j->gate || !dgate) &&
                     (j->scale || !dscale),
                 RWKV_E_NULL, "join_bwd: the gradient of a part that is not there");
    RWKV_REQUIRE((uintptr_t)stats % 16 == 0, RWKV_E_SHAPE, "join_bwd: misaligned stats");
    RWKV_REQUIRE(drop_ok(&j->drop), RWKV_E_UNSUPPORTED, "join_bwd: threshold %d of 65536", j->drop.threshold);
    void* const want[SUMS] = {dweight, dbias, dpost_weight, dpost_bias, dscale};
    JoinBwd a{xs, j->o, j->gate, j->ldo, j->ldg, stats, j->post_weight, j->post_bias, j->scale, j->weight,
              j->w_dt == RWKV_F32, dxs, dh, dx, dout, dgate, nullptr, {}, 0, j->N, (int)j->D, drop_of(j->drop)};
    Outs outs{};
    for (int k = 0; k < SUMS; ++k) {
        a.slot[k] = want[k] ? a.sums : -1;
        if (want[k]) outs.p[a.sums++] = want[k];
    }
    const int G = join_bwd_blocks(j->N, j->D);
    const int64_t need = (int64_t)G * a.sums * j->D * 4;
    RWKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), RWKV_E_SHAPE,
                 "join_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    if (a.sums) a.part = (float*)workspace;
    const hipStream_t s = (hipStream_t)stream;
    if (j->N > 0 && (a.sums || dx || dout || dgate)) {
        by_types(j->x_dt, j->dt, [&](auto ts, auto t) {
            by_width(j->D, [&](auto tpr) {
                constexpr int TPR = decltype(tpr)::value;
                rwkv::launch(join_bwd_kernel<decltype(ts), decltype(t), TPR>, dim3((unsigned)G), dim3(TPR == 64 ? 256 : TPR), s, a);
            });
        });
    }
    if (a.sums) {
        const dim3 grid((unsigned)((j->D + 15) / 16), (unsigned)a.sums);
        by_types(j->w_dt, j->w_dt, [&](auto, auto t) {
            rwkv::launch(join_reduce_kernel<decltype(t)>, grid, dim3(256), s, (const float*)workspace, G, a.sums, (int)j->D, outs);
        });
    }
    return status_of("join_bwd launch");
}

#define RWKV_TAIL_REQUIRE(what)                                                                                       \
    RWKV_REQUIRE(j, RWKV_E_NULL, what ": null arguments");                                                            \
    RWKV_REQUIRE(rwkv::dtype_ok(j->dt) && (j->o_dt == j->dt || j->o_dt == RWKV_F32) &&                                \
                     (j->w_dt == RWKV_F32 || j->w_dt == j->dt),                                                       \
                 RWKV_E_DTYPE, what ": types o %d, r %d, vectors %d", (int)j->o_dt, (int)j->dt, (int)j->w_dt);        \
    RWKV_REQUIRE(j->N >= 0 && j->N <= (1 << 24) && j->H >= 1 && j->H <= 1024 && j->ldo >= HEAD * j->H &&              \
                     j->ldr >= HEAD * j->H && j->ldk >= HEAD * j->H && j->ldv >= HEAD * j->H && j->ldg >= HEAD * j->H, \
                 RWKV_E_SHAPE, what ": N=%lld H=%lld (H <= 1024), or a pitch under 64 H", (long long)j->N,            \
                 (long long)j->H);                                                                                    \
    RWKV_REQUIRE(j->N == 0 || (j->o && j->r && j->k && j->v && j->gate && j->r_k && j->weight && j->bias),            \
                 RWKV_E_NULL, what ": null buffer")

rwkv_status rwkv_tail_fwd(const rwkv_tail* j, void* y, void* stream) {
    RWKV_TAIL_REQUIRE("tail_fwd");
    RWKV_REQUIRE(j->N == 0 || y, RWKV_E_NULL, "tail_fwd: null buffer");
    if (j->N == 0) return RWKV_OK;
    TailArgs a{};
    a.o = j->o, a.r = j->r, a.k = j->k, a.v = j->v, a.g = j->gate;
    a.ldo = j->ldo, a.ldr = j->ldr, a.ldk = j->ldk, a.ldv = j->ldv, a.ldg = j->ldg;
    a.rk = j->r_k, a.w = j->weight, a.b = j->bias, a.w32 = j->w_dt == RWKV_F32;
    a.y = y, a.N = j->N, a.C = (int)(HEAD * j->H), a.eps = j->eps;
    int TX, gx, gy;
    tail_geometry(a.N, a.C, TAIL_FWD_BLOCKS, TX, gx, gy);
    by_types(j->o_dt, j->dt, [&](auto to, auto t) {
        rwkv::launch(tail_fwd_kernel<decltype(to), decltype(t)>, dim3((unsigned)gx, (unsigned)gy), dim3(256),
                     (hipStream_t)stream, a, TX);
    });
    return status_of("tail_fwd launch");
}

int64_t rwkv_tail_bwd_workspace(int64_t N, int64_t H) {
    if (N < 0 || H < 1 || H > 1024) return 0;
    int TX, gx, gy;
    tail_geometry(N, HEAD * H, TAIL_BWD_BLOCKS, TX, gx, gy);
    return (int64_t)gy * 3 * HEAD * H * 4;
}

rwkv_status rwkv_tail_bwd(const rwkv_tail* j, const void* dy, int64_t lddy, void* dout, void* dr, void* dk, void* dv,
                          void* dgate, void* dr_k, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes,
                          void* stream) {
    RWKV_TAIL_REQUIRE("tail_bwd");
    RWKV_REQUIRE(j->N == 0 || dy, RWKV_E_NULL, "tail_bwd: null buffer");
    RWKV_REQUIRE(lddy >= HEAD * j->H, RWKV_E_SHAPE, "tail_bwd: lddy=%lld", (long long)lddy);
    const bool sums = dr_k || dweight || dbias;
    RWKV_REQUIRE(!sums || (dr_k && dweight && dbias), RWKV_E_NULL, "tail_bwd: dr_k, dweight and dbias go together");
    const int64_t need = sums ? rwkv_tail_bwd_workspace(j->N, j->H) : 0;
    RWKV_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), RWKV_E_SHAPE,
                 "tail_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    TailArgs a{};
    a.o = j->o, a.r = j->r, a.k = j->k, a.v = j->v, a.g = j->gate;
    a.ldo = j->ldo, a.ldr = j->ldr, a.ldk = j->ldk, a.ldv = j->ldv, a.ldg = j->ldg;
    a.rk = j->r_k, a.w = j->weight, a.b = j->bias, a.w32 = j->w_dt == RWKV_F32;
    a.dy = dy, a.lddy = lddy, a.dout = dout, a.dr = dr, a.dk = dk, a.dv = dv, a.dg = dgate;
    a.part = sums ? (float*)workspace : nullptr;
    a.N = j->N, a.C = (int)(HEAD * j->H), a.eps = j->eps;
    const hipStream_t s = (hipStream_t)stream;
    int TX, gx, gy;
    tail_geometry(a.N, a.C, TAIL_BWD_BLOCKS, TX, gx, gy);
    if (a.N > 0)
        by_types(j->o_dt, j->dt, [&](auto to, auto t) {
            rwkv::launch(tail_bwd_kernel<decltype(to), decltype(t)>, dim3((unsigned)gx, (unsigned)gy), dim3(256), s, a, TX);
        });
    if (sums) {
        const Outs outs{{dr_k, dweight, dbias, nullptr, nullptr}};
        const dim3 grid((unsigned)((a.C + 15) / 16), 3);
        by_types(j->w_dt, j->w_dt, [&](auto, auto t) {
            rwkv::launch(join_reduce_kernel<decltype(t)>, grid, dim3(256), s, (const float*)workspace, a.N > 0 ? gy : 0, 3, a.C, outs);
        });
    }
    return status_of("tail_bwd launch");
}

}  // extern "C"
