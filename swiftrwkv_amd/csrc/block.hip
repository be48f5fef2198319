// What a training block does around its recurrence and products, each in one
// pass over the rows: dropout from a counter-based generator, the join of one
// block with the next (norm, gate, dropout and scale of the branch, the
// residual sum, the next norm), and the recurrence's tail (head norm, bonus,
// gate) with its gradients.  The reference has the tail, the residual sum and
// the next norm, from MLX operations (RWKVBlock.swift:163-307); dropout and
// what may stand before the sum in a join are for blocks beside its own.
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

// 1/sqrt of a variance, to one step of fp32.  The hardware's takes a subnormal for
// zero (rows under 2^-63 with an eps of 0): those go in 2^64 times as large.
__device__ __forceinline__ float rstd_of(float x) {
    const bool small = x < 0x1p-126f;
    const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p64f : x);
    return small ? r * 0x1p32f : r;
}

// ───────────────────────────── chunks ─────────────────────────────

// How a row of D columns falls into chunks of eight: WHOLE, D is a multiple of 8;
// ENDS, it is not; FEW, D is under 8.
enum { WHOLE, ENDS, FEW };

// Eight values that were loaded `moved` columns before their place, into it:
// zeros from `valid` on.
__device__ __forceinline__ void move8(float (&v)[8], int moved, int valid) {
#pragma unroll
    for (int k = 4; k >= 1; k /= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (moved & k) v[i] = i + k < 8 ? v[i + k < 8 ? i + k : 7] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? v[i] : 0.0f;
}

// ───────────────────────────── dropout ─────────────────────────────

struct DropoutArgs {
    const void* x;
    const void* res;     // of y's type, or null
    void* y;             // [N, D]
    uint32_t ldx, ldr;
    int64_t chunks;      // N·cpr
    int cpr, D;          // chunks of 8 a row
    uint32_t magic;      // ceil(2^32 / cpr) where cpr is at most a block's chunks
    Drop drop;
};

// Chunks of 8 values, U a thread, a block's in one run; its first row is found
// once (in 64 bits), the others from there: a quotient under 2·RUN by a divisor
// of at most RUN is the high half of a 32-bit product with ceil(2^32 / cpr), and
// an address one product of 32 x 32 bits (products are a quarter of the rate of
// other operations, and the generator has 20 of them a chunk).  A chunk that
// passes its row's end is loaded as the row's last eight columns (FEW: one by
// one), and moved.
//
// Bound by bytes, and with 4 a value by the generator too: 32768 x 4096 bf16
// with an fp32 residual 235 us (5.7 TB/s), fp32 into bf16 143, bf16 96 (5.6).
constexpr int DROP_U = 4, DROP_RUN = 256 * DROP_U;

template <typename TX, typename TY, int ROWS>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const int64_t first = (int64_t)blockIdx.x * DROP_RUN;
    const int64_t row0 = first / a.cpr;
    const uint32_t rem = (uint32_t)(first - row0 * a.cpr);
    const int left = (int)min(a.chunks - first, (int64_t)DROP_RUN);
    const uint64_t key = a.drop.key();
    const TX* const x0 = reinterpret_cast<const TX*>(a.x) + row0 * a.ldx;
    const TY* const r0 = reinterpret_cast<const TY*>(a.res) + row0 * a.ldr;
    TY* const y0 = reinterpret_cast<TY*>(a.y) + row0 * a.D;
    Raw8<TX> x[DROP_U];
    Raw8<TY> r[DROP_U];
    uint32_t row[DROP_U], col[DROP_U];   // from row0; the chunk's first column
    auto valid = [&](int u) { return ROWS == WHOLE ? 8 : a.D - (int)col[u]; };
    auto load = [&](auto& r, auto* p, uint32_t ld, int u) {
        if constexpr (ROWS == FEW) r.load(p + (uint64_t)row[u] * ld, a.D);
        else __builtin_memcpy(r.q, p + ((uint64_t)row[u] * ld + (ROWS == ENDS ? min(col[u], (uint32_t)a.D - 8) : col[u])), sizeof(r.q));
    };
    auto get = [&](const auto& r, int u, float (&v)[8]) {
        r.get(v);
        if constexpr (ROWS == ENDS)
            if (valid(u) < 8) move8(v, 8 - valid(u), valid(u));
    };
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
        // (threads behind the last chunk have it again)
        const uint32_t n = rem + min((int)threadIdx.x + 256 * u, left - 1);
        row[u] = a.cpr == 1 ? n : a.cpr > DROP_RUN ? (n >= (uint32_t)a.cpr) : __umulhi(n, a.magic);
        col[u] = 8 * (n - row[u] * a.cpr);
        load(x[u], x0, a.ldx, u);
        if (a.res) load(r[u], r0, a.ldr, u);
    }
#pragma unroll
    for (int u = 0; u < DROP_U; ++u) {
        if ((int)threadIdx.x + 256 * u >= left) continue;
        float v[8], m[8];
        get(x[u], u, v);
        if (a.drop.threshold) {
            factors(a.drop, key, col[u] / 8, (uint32_t)row0 + row[u], m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = dropped(m[i], v[i]);
        }
        if (a.res) {
            get(r[u], u, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += m[i];
        }
        store8(y0 + ((uint64_t)row[u] * (uint32_t)a.D + col[u]), valid(u), v);
    }
}

// ───────────────────────────── join ─────────────────────────────

// Sum over the TPR lanes of a row: sixteen, or a wave.
template <int TPR>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (TPR != 16) return rwkv_wkv::wave_total(x);
    auto turned = [](float v, auto ctrl) {
        return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    x = turned(x, std::integral_constant<int, 0x128>{});   // row_ror:8, 4, 2, 1
    x = turned(x, std::integral_constant<int, 0x124>{});
    x = turned(x, std::integral_constant<int, 0x122>{});
    return turned(x, std::integral_constant<int, 0x121>{});
}

// Sums over the TPR threads of a row, of one value or two, as the layer norm
// takes one: its lanes, or the block through LDS, the waves in order.  Every
// thread has read a slot before the barrier of the next sum, so two slots in
// turn are enough.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float s, float q, float2 (*part)[16], int slot) {
    s = lanes_sum<TPR>(s);
    q = lanes_sum<TPR>(q);
    if constexpr (TPR <= 64) {
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
    s = lanes_sum<TPR>(s);
    if constexpr (TPR <= 64) {
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

// A thread's eight columns of a row.  Threads whose chunk passes the row's end,
// or lies behind it, load the row's last eight columns, unconditionally (FEW:
// one by one), and move them into place where they are used; WHOLE has none of
// the former, and what the latter make of their load goes nowhere.  (Loads that
// look at every value, in the same kernel, cost half of its time in branches
// and moves.)
template <int ROWS>
struct Cols {
    int col, valid;   // first column, and columns from there to the row's end
    int at;           // where the thread loads
    __device__ __forceinline__ Cols(int t, int D) : col(8 * t), valid(D - 8 * t), at(ROWS == FEW ? 8 * t : min(8 * t, D - 8)) {}
    // A row's value at: a row's address is the same for all and stays in scalar
    // registers, under a 32-bit offset of the thread's.
    template <typename T>
    static __device__ __forceinline__ T* place(T* row, int at) {
        using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
        uint32_t off = (uint32_t)(at * (int)sizeof(T));
        asm volatile("" : "+v"(off));   // (else the compiler keeps 64-bit addresses of every tensor over the loop)
        return reinterpret_cast<T*>(reinterpret_cast<Byte*>(row) + off);
    }
    // value i is one of the row's; of a sum, whether the thread has any
    __device__ __forceinline__ bool has(int i) const { return ROWS == WHOLE || i < valid; }
    __device__ __forceinline__ float own(float s) const { return ROWS != WHOLE || valid > 0 ? s : 0.0f; }
    template <typename T>
    __device__ __forceinline__ void load(Raw8<T>& r, const void* p, int64_t row, int64_t ld) const {
        const T* q = place(reinterpret_cast<const T*>(p) + row * ld, at);
        if constexpr (ROWS == FEW) r.load(q, valid);
        else __builtin_memcpy(r.q, q, sizeof(r.q));
    }
    // The values loaded, zeros past the row's end (WHOLE: any).
    template <typename T>
    __device__ __forceinline__ void get(Raw8<T> r, float (&v)[8]) const {
        if constexpr (ROWS != ENDS) return r.get(v);
        r.get(v);
        if (col != at) move8(v, col - at, valid);
    }
    template <typename T>
    __device__ __forceinline__ void store(void* p, int64_t row, int D, const float (&v)[8]) const {
        if (valid > 0) store8(place(reinterpret_cast<T*>(p) + row * D, col), ROWS == WHOLE ? 8 : valid, v);
    }
    // The vector w's values of the columns, or `otherwise` without one.
    template <typename T>
    __device__ __forceinline__ void vector(const void* w, int w32, float otherwise, float (&v)[8]) const {
        const int from = ROWS == WHOLE ? at : col, n = ROWS == WHOLE ? 8 : valid;
        if (w && w32) load8(place(reinterpret_cast<const float*>(w), from), n, v);
        else if (w) load8(place(reinterpret_cast<const T*>(w), from), n, v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = otherwise;
    }
};

struct JoinFwd {
    const void *x, *o, *gate;   // gate, post_w, post_b, scale, b may be null
    int64_t ldx, ldo, ldg;
    const void *post_w, *post_b, *scale, *w, *b;
    int w32;                    // the vectors are fp32 (else o's type)
    void *xs, *h;               // [N, D]
    float* stats;               // [N, 4]: mean and rstd of o (0, 1 without its norm), of x'; or null
    int64_t N;
    int D;
    float post_eps, eps;
    Drop drop;
};

// A block's threads, its rows at a time, and the row that TPR of its threads
// begin with.
constexpr int threads_of(int tpr) { return tpr < 256 ? (tpr == 128 ? 128 : 256) : tpr; }
constexpr int rows_of(int tpr) { return threads_of(tpr) / tpr; }
template <int TPR>
__device__ __forceinline__ int64_t first_row() {
    if constexpr (TPR == 16) return (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    else if constexpr (TPR == 64) return (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    else return blockIdx.x;
}

// A chunk of eight equal values: what stands for a part that is not there, so
// that no value of a row has two ways to come about.
template <typename T>
__device__ __forceinline__ Raw8<T> filled(float x) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)x;
    Raw8<T> r;
    __builtin_memcpy(r.q, t, sizeof(r.q));
    return r;
}

// Rows first_row(), + gridDim.x·RPB, ...; a thread holds one chunk of 8 columns
// of a row, and the next row's is on its way.  Bound by bytes: 16384 x 2048, fp32
// stream, bf16 o and gate, every part: 90 us (5.2 TB/s; a large copy 5.1); a bf16
// stream 65 (5.1), and without gate, post norm, scale and dropout 43.  With the
// next row's loads under a choice, 64-bit addresses and a look at every value of a
// chunk the first took 112.
template <typename TS, typename T, int TPR, int ROWS>
__global__ __launch_bounds__(threads_of(TPR)) void join_fwd_kernel(JoinFwd a) {
    __shared__ float2 part[2][16];
    const int t = threadIdx.x % TPR;
    const Cols<ROWS> c(t, a.D);
    const int64_t step = (int64_t)gridDim.x * rows_of(TPR);
    int64_t row = first_row<TPR>();
    if (row >= a.N) return;   // rows that share a barrier end together
    const float per = 1.0f / (float)a.D;
    const uint64_t key = a.drop.threshold ? a.drop.key() : 0;
    Raw8<TS> rx;
    Raw8<T> ro, rg = filled<T>(1.0f);
    auto load = [&](int64_t r) {
        c.load(ro, a.o, r, a.ldo);
        c.load(rx, a.x, r, a.ldx);
        if (a.gate) c.load(rg, a.gate, r, a.ldg);
    };
    load(row);
    float pw[8], pb[8], sc[8], w[8], b[8];
    c.template vector<T>(a.post_w, a.w32, 1.0f, pw);
    c.template vector<T>(a.post_b, a.w32, 0.0f, pb);
    c.template vector<T>(a.scale, a.w32, 1.0f, sc);
    c.template vector<T>(a.w, a.w32, 1.0f, w);
    c.template vector<T>(a.b, a.w32, 0.0f, b);
    for (; row < a.N; row += step) {
        float v[8], u[8], g[8];
        c.get(ro, u);
        c.get(rx, v);
        c.get(rg, g);
        load(min(row + step, a.N - 1));   // (the last row again rather than a choice)
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
        if (a.post_w) {
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += u[i];
            st.x = row_sum<TPR>(c.own(s), part, 0) * per;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[i] -= st.x;
                q += c.has(i) ? u[i] * u[i] : 0.0f;
            }
            st.y = rstd_of(row_sum<TPR>(c.own(q), part, 1) * per + a.post_eps);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = (u[i] * st.y * pw[i] + pb[i]) * g[i];
        if (a.drop.threshold) {
            factors(a.drop, key, (uint32_t)t, (uint32_t)row, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = dropped(g[i], u[i]);
        }
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = c.has(i) ? v[i] + sc[i] * u[i] : 0.0f;
            s += v[i];
        }
        c.template store<TS>(a.xs, row, a.D, v);
        st.z = row_sum<TPR>(c.own(s), part, 0) * per;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] -= st.z;
            q += c.has(i) ? v[i] * v[i] : 0.0f;
        }
        st.w = rstd_of(row_sum<TPR>(c.own(q), part, 1) * per + a.eps);
        if (a.stats && t == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = st;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * st.w * w[i] + b[i];
        c.template store<T>(a.h, row, a.D, v);
    }
}

enum { DW, DB, DPW, DPB, DSC, SUMS };   // column sums of the join, the scale's last

struct JoinBwd {
    const void *xs, *o, *gate;  // x', or x where x' has 16 bits; o null: it does not reach a gradient
    int64_t ldx, ldo, ldg;
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

// N times eight values of a thread in LDS slots that it alone writes and reads.
template <int N, int THREADS>
struct Slots {
    float4 (&v)[2 * N][THREADS];
    __device__ __forceinline__ void put(int k, const float (&x)[8]) const {
        v[2 * k][threadIdx.x] = make_float4(x[0], x[1], x[2], x[3]);
        v[2 * k + 1][threadIdx.x] = make_float4(x[4], x[5], x[6], x[7]);
    }
    __device__ __forceinline__ void get(int k, float (&x)[8]) const {
        const float4 a = v[2 * k][threadIdx.x], b = v[2 * k + 1][threadIdx.x];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};

// With xh = (x' − μ)·r and G the whole gradient of x':
//   G = dx' + LN'(dh·w; xh, r), dw = Σ dh·xh, db = Σ dh
//   du = G·s·m, ds = Σ G·m·u, dg = du·n, dn = du·g
//   do = LN'(dn·w1; oh, r1), dw1 = Σ dn·oh, db1 = Σ dn
// LN'(y; h, r) = r·(y − mean y − h·mean(y·h)).
//
// A stream of 16 bits holds x' rounded, which would put that rounding into xh and
// so into sums of fp32: x' is formed again from x, o and the gate, which are read
// anyway.
//
// A chunk is loaded as soon as the one before it has been taken apart, so the
// next row is on its way under this one's two sums over the row.  The vectors
// lie in LDS.  The sizes above, back to back and with the sums' join, 6 us of it: 145
// us (5.1 TB/s), a bf16 stream 114 (4.7); without gate, post norm, scale and dropout
// 112 (4.8) and 82 (4.9).  With three waves a SIMD instead of two, by launch bounds,
// registers spilled (327 us where two took 197).  With 1024 threads, which have 128
// registers each, the column sums lie in LDS instead, and the vectors and rows are
// read where they are used: 4096 x 8192 184 us.
template <typename TS, typename T, int TPR, int ROWS>
__global__ __launch_bounds__(threads_of(TPR)) void join_bwd_kernel(JoinBwd a) {
    constexpr int RPB = rows_of(TPR);
    __shared__ float2 part[2][16];
    __shared__ float sums[RPB > 1 ? 8 * 256 : 1];
    __shared__ float4 slots[8][threads_of(TPR)];
    constexpr bool AHEAD = TPR < 1024, AGAIN = sizeof(TS) == 2;   // rows read ahead; x' formed again
    enum { PW, PB, SC, W };
    const Slots<4, threads_of(TPR)> lds{slots};
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const Cols<ROWS> at(t, a.D);
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float per = 1.0f / (float)a.D;
    const uint64_t key = a.drop.threshold ? a.drop.key() : 0;
    Raw8<TS> rdx = filled<TS>(0.0f), rx;
    Raw8<T> rdh, ro = filled<T>(0.0f), rg = filled<T>(1.0f);
    auto load_h = [&](int64_t r) {
        if (!a.dh) return;
        at.load(rdh, a.dh, r, a.D);
        at.load(rx, a.xs, r, a.ldx);
    };
    auto load_o = [&](int64_t r) {
        if constexpr (!AHEAD) rdx = filled<TS>(0.0f), ro = filled<T>(0.0f), rg = filled<T>(1.0f);   // (not kept from row to row)
        if (a.dxs) at.load(rdx, a.dxs, r, a.D);
        if (a.o) at.load(ro, a.o, r, a.ldo);
        if (a.gate) at.load(rg, a.gate, r, a.ldg);
    };
    int64_t row = first_row<TPR>();
    float4 next = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (AHEAD && row < a.N) {
        next = *reinterpret_cast<const float4*>(a.stats + 4 * row);
        load_h(row);
        load_o(row);
    }
    const void* const vectors[4] = {a.post_w, a.post_b, a.scale, a.w};
    auto vector = [&](int k, float (&x)[8]) {   // or, of a missing one, what changes nothing
        if constexpr (AHEAD) lds.get(k, x);
        else at.template vector<T>(vectors[k], a.w32, k == PB ? 0.0f : 1.0f, x);
    };
    float acc[SUMS][8] = {};
    auto add = [&](int k, const float (&x)[8]) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[k][i] += x[i];
        } else {
            float s[8];
            lds.get(k, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += x[i];
            lds.put(k, s);
        }
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float x[8] = {};
        if constexpr (AHEAD) at.template vector<T>(vectors[k], a.w32, k == PB ? 0.0f : 1.0f, x);
        lds.put(k, x);
    }
    int slot = 0;
    for (; row < a.N; row += step) {
        const int64_t then = min(row + step, a.N - 1);   // (the last row again rather than a choice)
        const float4 st = AHEAD ? next : *reinterpret_cast<const float4*>(a.stats + 4 * row);
        if constexpr (!AHEAD) load_h(row);
        float G[8], y[8], c[8], oh[8], nv[8];
        if constexpr (AHEAD) next = *reinterpret_cast<const float4*>(a.stats + 4 * then);
        // oh, n, the gate and, where something is dropped, m
        float m[8];
        auto branch = [&](float (&gate)[8]) {
            if constexpr (!AHEAD) {
                __builtin_amdgcn_sched_barrier(0);   // (not ahead: registers)
                load_o(row);
            }
            float b[8];
            at.get(ro, oh);
            at.get(rg, gate);
            vector(PW, c);
            vector(PB, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                oh[i] = at.has(i) ? (oh[i] - st.x) * st.y : 0.0f;
                nv[i] = oh[i] * c[i] + b[i];
            }
            if (a.drop.threshold) factors(a.drop, key, (uint32_t)t, (uint32_t)row, m);
        };
        float gate[8], sc[8];
        if constexpr (AGAIN) {
            branch(gate);
            vector(SC, sc);
        }
        if (a.dh) {
            float xh[8];
            at.get(rdh, y);
            at.get(rx, xh);
            if constexpr (AHEAD) load_h(then);
            if constexpr (AGAIN) {   // as the forward pass forms x'
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float u = nv[i] * gate[i];
                    if (a.drop.threshold) u = dropped(m[i], u);
                    xh[i] = at.has(i) ? xh[i] + sc[i] * u : 0.0f;
                }
            }
            add(DB, y);
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                xh[i] = at.has(i) ? (xh[i] - st.z) * st.w : 0.0f;
                c[i] = y[i] * xh[i];
            }
            add(DW, c);
            vector(W, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] *= c[i];
                s1 += y[i];
                s2 += y[i] * xh[i];
            }
            const float2 s = row_sum2<TPR>(at.own(s1), at.own(s2), part, slot);
            slot ^= 1;
            s1 = s.x * per, s2 = s.y * per;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (y[i] - s1 - xh[i] * s2) * st.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = 0.0f;
        }
        if constexpr (!AGAIN) branch(gate);
        at.get(rdx, G);
#pragma unroll
        for (int i = 0; i < 8; ++i) G[i] += y[i];
        if (a.dx) at.template store<TS>(a.dx, row, a.D, G);
        if constexpr (AHEAD) load_o(then);
        float u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            u[i] = gate[i] * nv[i];
            y[i] = gate[i];
            G[i] = at.has(i) ? G[i] : 0.0f;   // (not zero of itself past the row's end)
        }
        if (a.drop.threshold) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[i] = dropped(m[i], u[i]);   // m of G, for the sum
                nv[i] = dropped(m[i], nv[i]);
                y[i] = dropped(m[i], y[i]);
                G[i] = m[i] > 0.0f ? G[i] : 0.0f;   // (zeros times an infinity are none)
            }
        }
        if constexpr (!AGAIN) vector(SC, sc);
        vector(PW, c);
        float p1 = 0.0f, p2 = 0.0f;
        // u: dn·oh; y: dn; nv: dg; G: dn·w1
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            acc[DSC][i] += G[i] * u[i];
            G[i] *= sc[i];
            nv[i] *= G[i];
            y[i] *= G[i];
            u[i] = y[i] * oh[i];
            G[i] = y[i] * c[i];
            p1 += G[i];
            p2 += G[i] * oh[i];
        }
        add(DPB, y);
        add(DPW, u);
        if (a.dgate) at.template store<T>(a.dgate, row, a.D, nv);
        if (!a.dout) continue;
        if (a.post_w) {
            const float2 p = row_sum2<TPR>(at.own(p1), at.own(p2), part, slot);
            slot ^= 1;
            p1 = p.x * per, p2 = p.y * per;
#pragma unroll
            for (int i = 0; i < 8; ++i) G[i] = (G[i] - p1 - oh[i] * p2) * st.y;
        }
        at.template store<T>(a.dout, row, a.D, G);
    }
    if (!a.part) return;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        if (a.slot[k] < 0) continue;   // the same for all
        if constexpr (!AHEAD)
            if (k != DSC) lds.get(k, acc[k]);
        if constexpr (RPB > 1) {
            // the block's row groups meet in order
            __syncthreads();
            if (grp > 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[(grp * 8 + i) * TPR + t] = acc[k][i];
            __syncthreads();
            if (grp == 0)
                for (int r = 1; r < RPB; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[k][i] += sums[(r * 8 + i) * TPR + t];
        }
        if (grp == 0) at.template store<float>(a.part, (int64_t)blockIdx.x * a.sums + a.slot[k], a.D, acc[k]);
    }
}

struct Outs {
    void* p[SUMS];
};

// Column sums of part [G][sums][D] (G may be 0) into out.p[0 .. sums): a block
// owns 32 columns (a cache line) of one sum and splits the G rows over 32 thread
// rows, each in order, whose loads are all on their way at once up to 512; the 32
// partial sums meet in LDS, by halves.
template <typename T>
__global__ __launch_bounds__(1024) void join_reduce_kernel(const float* part, int G, int sums, int D, Outs out) {
    __shared__ float s[32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, k = blockIdx.y;
    const int col = min((int)blockIdx.x * 32 + c, D - 1);
    float t = 0.0f;
#pragma unroll 16
    for (int g = r; g < G; g += 32) t += part[((int64_t)g * sums + k) * D + col];
    s[r][c] = t;
    __syncthreads();
    t = s[c][r];   // row c's sum of column r
#pragma unroll
    for (int h = 16; h >= 1; h /= 2) t += __shfl_xor(t, h);
    const int at = blockIdx.x * 32 + r;
    if (c != 0 || at >= D) return;
    T* o = reinterpret_cast<T*>(out.p[0]);
#pragma unroll
    for (int i = 1; i < SUMS; ++i)
        if (k == i) o = reinterpret_cast<T*>(out.p[i]);
    o[at] = (T)t;
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
// rows down a block, rows strided over gridDim.y, the next one on its way.
// Bound by bytes: 32768 x 32 heads, o fp32, the rest bf16: 186 us back to back
// (5.05 TB/s; a large copy 5.1), 200 between a training pass's other kernels.
template <typename TO, typename T>
__global__ __launch_bounds__(256) void tail_fwd_kernel(TailArgs a, int TX) {
    const int tx = threadIdx.x % TX, col = 8 * (blockIdx.x * TX + tx);
    if (col >= a.C) return;   // whole heads
    const int64_t step = (int64_t)gridDim.y * (256 / TX);
    float rk[8], w[8], b[8];
    load_w<T>(a.rk, a.w32, col, 8, rk);
    load_w<T>(a.w, a.w32, col, 8, w);
    load_w<T>(a.b, a.w32, col, 8, b);
    int64_t row = (int64_t)blockIdx.y * (256 / TX) + threadIdx.x / TX;
    if (row >= a.N) return;
    Raw8<TO> ro;
    Raw8<T> rr, rkk, rv, rg;
    auto load = [&](int64_t at) {
        ro.load(reinterpret_cast<const TO*>(a.o) + at * a.ldo + col, 8);
        rr.load(reinterpret_cast<const T*>(a.r) + at * a.ldr + col, 8);
        rkk.load(reinterpret_cast<const T*>(a.k) + at * a.ldk + col, 8);
        rv.load(reinterpret_cast<const T*>(a.v) + at * a.ldv + col, 8);
        rg.load(reinterpret_cast<const T*>(a.g) + at * a.ldg + col, 8);
    };
    load(row);
    for (; row < a.N; row += step) {
        float o[8], r[8], k[8], v[8], g[8];
        ro.get(o);
        rr.get(r);
        rkk.get(k);
        rv.get(v);
        rg.get(g);
        load(min(row + step, a.N - 1));
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
        const float inv = rstd_of(sum8(q) * (1.0f / HEAD) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (o[i] * inv * w[i] + b[i] + d * v[i]) * g[i];
        store8(reinterpret_cast<T*>(a.y) + row * a.C + col, 8, o);
    }
}

// With oh = (o − μ)·i, d = Σ r·k·r_k, q = oh·w + b + d·v:
//   dg = dy·q, dq = dy·g, dv = dq·d, e = Σ dq·v, dr = e·k·r_k, dk = e·r·r_k
//   do = LN'(dq·w; oh, i);  dr_k = Σ e·r·k, dw = Σ dq·oh, db = Σ dq
// μ and i are formed again: o is read anyway.  Bound by bytes, 26 a value: the
// same sizes in 313 us (5.6 TB/s) and 5 of the sums' join in a training pass, 324
// for both back to back.
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
            const float inv = rstd_of(sum8(q) * (1.0f / HEAD) + a.eps);
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

// Threads of a row, and how it falls into chunks.
template <typename F>
void by_width(int64_t D, F f) {
    auto by_ends = [&](auto tpr) {
        if (D % 8 == 0) f(tpr, std::integral_constant<int, WHOLE>{});
        else f(tpr, std::integral_constant<int, ENDS>{});
    };
    if (D < 8) f(std::integral_constant<int, 16>{}, std::integral_constant<int, FEW>{});
    else if (D <= 128) by_ends(std::integral_constant<int, 16>{});
    else if (D <= 512) by_ends(std::integral_constant<int, 64>{});
    else if (D <= 1024) by_ends(std::integral_constant<int, 128>{});
    else if (D <= 2048) by_ends(std::integral_constant<int, 256>{});
    else if (D <= 4096) by_ends(std::integral_constant<int, 512>{});
    else by_ends(std::integral_constant<int, 1024>{});
}

// Blocks of the join's passes: what the registers of 256 CUs hold at once (rows
// beyond are walked).
int64_t join_rows_at_once(int64_t D) { return D <= 128 ? 16 : D <= 512 ? 4 : 1; }
int join_fwd_blocks(int64_t N, int64_t D) {
    const int full = D <= 512 ? 1024 : D <= 1024 ? 2048 : D <= 2048 ? 1024 : D <= 4096 ? 512 : 256;
    const int64_t rpb = join_rows_at_once(D);
    return (int)std::min<int64_t>((N + rpb - 1) / rpb, full);
}
// What the registers hold, each block writing one partial row per column sum; and
// from 256 blocks on no more than one for four of its rows.  us of the backward
// pass by 256, 512 and 768 blocks (fp32 stream, bf16, every part): 600 x 2048 18.8,
// 20.7, 24.7; 2048 x 2048 27.0, 26.4, 33.3; 16384 x 2048 160, 146, 172.  (Measured at
// 2048 columns with every part alone, and taken over for the others.)
int join_bwd_blocks(int64_t N, int64_t D) {
    const int64_t full = D <= 512 ? 512 : D <= 1024 ? 1024 : D <= 2048 ? 512 : 256;
    const int64_t blocks = (N + join_rows_at_once(D) - 1) / join_rows_at_once(D);
    return (int)std::min({blocks, full, std::max<int64_t>(256, blocks / 4)});
}

// Lanes across and the grid of the tail's passes.
void tail_geometry(int64_t N, int64_t C, int most, int& TX, int& gx, int& gy) {
    const int64_t chunks = C / 8;
    TX = 64;
    // no more than an eighth of the lanes beyond the last head
    while (TX > 8 && ((chunks + TX - 1) / TX * TX - chunks) * 8 > chunks) TX /= 2;
    gx = (int)((chunks + TX - 1) / TX);
    const int ty = 256 / TX;
    gy = (int)std::max<int64_t>(1, std::min<int64_t>((N + ty - 1) / ty, std::max(1, most / gx)));
}
// (32768 x 32 heads: forward 183 us by 512 blocks, 186 by 1024, 185 by 4096, a few
// rows 7.7 and 6.6; backward 330 by 512, whose partial rows are half of 1024's 342)
constexpr int TAIL_FWD_BLOCKS = 1024, TAIL_BWD_BLOCKS = 512;

bool join_ok(const rwkv_join* a) {
    return (a->x_dt == a->dt || a->x_dt == RWKV_F32) && rwkv::dtype_ok(a->dt) && (a->w_dt == RWKV_F32 || a->w_dt == a->dt);
}

}  // namespace

extern "C" {

rwkv_status rwkv_dropout(const void* x, rwkv_dtype x_dt, int64_t ldx, const void* residual, int64_t ldr, void* y,
                         rwkv_dtype y_dt, const rwkv_drop* drop, int64_t N, int64_t D, void* stream) {
    RWKV_REQUIRE(pair_ok(x_dt, y_dt), RWKV_E_DTYPE, "dropout: types x %d, y %d", (int)x_dt, (int)y_dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= (1 << 22) && ldx >= D && ldx <= RWKV_DROPOUT_MAX_PITCH &&
                     (!residual || (ldr >= D && ldr <= RWKV_DROPOUT_MAX_PITCH)),
                 RWKV_E_SHAPE, "dropout: N=%lld D=%lld ldx=%lld ldr=%lld", (long long)N, (long long)D, (long long)ldx, (long long)ldr);
    RWKV_REQUIRE(N == 0 || (x && y), RWKV_E_NULL, "dropout: null buffer");
    RWKV_REQUIRE(drop_ok(drop), RWKV_E_UNSUPPORTED, "dropout: threshold %d of 65536", drop ? drop->threshold : -1);
    if (N == 0) return RWKV_OK;
    const int64_t cpr = (D + 7) / 8, chunks = N * cpr, blocks = (chunks + DROP_RUN - 1) / DROP_RUN;
    RWKV_REQUIRE(blocks < (int64_t(1) << 31), RWKV_E_SHAPE, "dropout: %lld values", (long long)(N * D));
    const DropoutArgs a{x, residual, y, (uint32_t)ldx, residual ? (uint32_t)ldr : 0u, chunks, (int)cpr, (int)D,
                        (uint32_t)(((uint64_t(1) << 32) + cpr - 1) / cpr), drop_of(*drop)};
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks);
    auto launch = [&](auto tx, auto ty) {
        if (D < 8) rwkv::launch(dropout_kernel<decltype(tx), decltype(ty), FEW>, grid, dim3(256), s, a);
        else if (D % 8 == 0) rwkv::launch(dropout_kernel<decltype(tx), decltype(ty), WHOLE>, grid, dim3(256), s, a);
        else rwkv::launch(dropout_kernel<decltype(tx), decltype(ty), ENDS>, grid, dim3(256), s, a);
    };
    if (y_dt == RWKV_F32 || x_dt == y_dt) by_types(y_dt, x_dt, [&](auto ty, auto tx) { launch(tx, ty); });
    else by_types(x_dt, y_dt, [&](auto tx, auto ty) { launch(tx, ty); });
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
        by_width(j->D, [&](auto tpr, auto ends) {
            constexpr int TPR = decltype(tpr)::value;
            rwkv::launch(join_fwd_kernel<decltype(ts), decltype(t), TPR, decltype(ends)::value>, grid, dim3(threads_of(TPR)),
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
    const bool again = j->x_dt != RWKV_F32;   // x' is formed again
    RWKV_REQUIRE(!again || !j->x || j->ldx >= j->D, RWKV_E_SHAPE, "join_bwd: ldx=%lld", (long long)j->ldx);
    RWKV_REQUIRE(j->N == 0 || ((again ? j->x && j->o : xs && (j->o || !(j->gate || j->post_weight || j->scale))) && j->weight && stats),
                 RWKV_E_NULL, "join_bwd: null buffer");
    RWKV_REQUIRE((j->post_weight || (!j->post_bias && !dpost_weight && !dpost_bias)) && (j->gate || !dgate) &&
                     (j->scale || !dscale),
                 RWKV_E_NULL, "join_bwd: the gradient of a part that is not there");
    RWKV_REQUIRE((uintptr_t)stats % 16 == 0, RWKV_E_SHAPE, "join_bwd: misaligned stats");
    RWKV_REQUIRE(drop_ok(&j->drop), RWKV_E_UNSUPPORTED, "join_bwd: threshold %d of 65536", j->drop.threshold);
    void* const want[SUMS] = {dweight, dbias, dpost_weight, dpost_bias, dscale};
    JoinBwd a{again ? j->x : xs, j->o, j->gate, again ? j->ldx : j->D, j->ldo, j->ldg, stats, j->post_weight, j->post_bias, j->scale, j->weight,
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
            by_width(j->D, [&](auto tpr, auto ends) {
                constexpr int TPR = decltype(tpr)::value;
                rwkv::launch(join_bwd_kernel<decltype(ts), decltype(t), TPR, decltype(ends)::value>, dim3((unsigned)G), dim3(threads_of(TPR)), s, a);
            });
        });
    }
    if (a.sums) {
        const dim3 grid((unsigned)((j->D + 31) / 32), (unsigned)a.sums);
        by_types(j->w_dt, j->w_dt, [&](auto, auto t) {
            rwkv::launch(join_reduce_kernel<decltype(t)>, grid, dim3(1024), s, (const float*)workspace, G, a.sums, (int)j->D, outs);
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
        const dim3 grid((unsigned)((a.C + 31) / 32), 3);
        by_types(j->w_dt, j->w_dt, [&](auto, auto t) {
            rwkv::launch(join_reduce_kernel<decltype(t)>, grid, dim3(1024), s, (const float*)workspace, a.N > 0 ? gy : 0, 3, a.C, outs);
        });
    }
    return status_of("tail_bwd launch");
}

}  // extern "C"
