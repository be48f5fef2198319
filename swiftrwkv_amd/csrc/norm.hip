// Layer norm with its gradients, and the 8-bit activation checkpoint
// (training around the recurrence; RWKVBlock's ln1 / ln2 / ln_out,
// Sources/RWKVModel/RWKVBlock.swift:163-307, which the reference differentiates
// through MLX's own layer norm).
//
//   μ = mean x, r = 1/√(mean (x−μ)² + ε), x̂ = (x−μ)·r, y = x̂·w + b
//   g = dy·w, dx = r·(g − mean g − x̂·mean(g·x̂)), dw = Σ_rows dy·x̂, db = Σ_rows dy
//
// All statistics, sums and gradients are fp32; one rounding per output.  The
// backward pass takes x itself or its 8-bit checkpoint (act8.h), with the
// forward's fp32 μ and r either way.
//
// Bound by bytes.  32768 × 4096 fp32 into bf16 with the row kept in 8 bits
// (943 MB each way): forward 179 µs (5.3 TB/s; a large copy 5.1), backward 274
// (3.4), its sums' join 9.  8192 × 2048 bf16 with fp32 weights: 18 µs, 34 and 5.
// The checkpoint alone, 16384 × 8192 bf16: 82 µs into 8 bits, 88 back (4.9, 4.6).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "act8.h"
#include "launch.h"
#include "wkv7_step.h"

namespace {

using namespace rwkv_train;
typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int MAX_D = 65536;

// ───────────────────────────── row reductions ─────────────────────────────

// Sum over the TPR threads of a row: one wave (TPR 64), or the whole block
// through LDS, every thread adding the waves in order.  `slot` alternates so
// that one barrier per sum is enough: a wave can be at most one sum ahead.
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float (*part)[16], int slot) {
    s = rwkv_wkv::wave_total(s);
    if constexpr (TPR == 64) {
        return s;
    } else {
        if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = s;
        __syncthreads();
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) t += part[slot][i];
        return t;
    }
}

struct NormFwd {
    const void* x;
    int64_t ldx;
    const void* w;
    const void* b;          // may be null
    int w32;                // w, b fp32 (else x's type)
    void* y;                // [N, D]
    float* stats;           // [N, 2]: mean, rstd; may be null
    int8_t* codes;          // [N, Dp] or null
    uint8_t* scales;        // [N, Dp/32]
    int64_t N;
    int D;
    float eps;
};

template <typename T>
__device__ __forceinline__ void load_w(const void* w, int w32, int col, int valid, float (&v)[8]) {
    if (w32)
        load8(reinterpret_cast<const float*>(w) + col, valid, v);
    else
        load8(reinterpret_cast<const T*>(w) + col, valid, v);
}

// TPR threads hold one row in registers, thread t the 8-value chunks
// t + TPR·j, j < NV, and walk the rows blockIdx.x·RPB + threadIdx.x / TPR,
// + gridDim.x·RPB, ...: up to 16384 columns w and b stay in registers from row
// to row (fp32 weights are four times a bf16 row's bytes) and the next row is
// loaded while one is worked on.
template <typename TX, typename TY, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_fwd_kernel(NormFwd a) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    constexpr bool HOLD = NV <= 4;
    __shared__ float part[2][16];
    const int t = threadIdx.x % TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= a.N) return;   // whole waves; no row shares a barrier where RPB > 1
    const TX* x = reinterpret_cast<const TX*>(a.x);
    const int64_t dp = padded(a.D);
    float w[HOLD ? NV : 1][8], b[HOLD ? NV : 1][8];
    Raw8<TX> next[NV];
    auto load_row = [&](int64_t r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) next[j].load(x + r * a.ldx + 8 * (t + TPR * j), a.D - 8 * (t + TPR * j));
    };
    if constexpr (HOLD) {
        load_row(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j);
            load_w<TX>(a.w, a.w32, col, a.D - col, w[j]);
            if (a.b) load_w<TX>(a.b, a.w32, col, a.D - col, b[j]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) b[j][i] = 0.0f;
        }
    }
    for (; row < a.N; row += step) {
        float v[NV][8];
        float s = 0.0f;
        if constexpr (!HOLD) load_row(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) next[j].get(v[j]);
        if (HOLD && row + step < a.N) load_row(row + step);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[j][i];
        const float mean = row_sum<TPR>(s, part, 0) / (float)a.D;
        float q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = v[j][i] - mean;
                q += col + i < a.D ? d * d : 0.0f;
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, part, 1) / (float)a.D + a.eps);
        if (a.stats && t == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mean, rstd);
        TY* yr = reinterpret_cast<TY*>(a.y) + row * a.D;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j), valid = a.D - col;
            if (a.codes && col < dp) {   // whole quads: dp is a multiple of 32
                uint32_t scale;
                const uint2 c = encode8(v[j], scale);
                *reinterpret_cast<uint2*>(a.codes + row * dp + col) = c;
                if ((t & 3) == 0) a.scales[(row * dp + col) / GROUP] = (uint8_t)scale;
            }
            if (valid <= 0) continue;
            float y[8];
            if constexpr (HOLD) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = (v[j][i] - mean) * rstd * w[j][i] + b[j][i];
            } else {
                load_w<TX>(a.w, a.w32, col, valid, w[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = (v[j][i] - mean) * rstd * w[0][i];
                if (a.b) {
                    load_w<TX>(a.b, a.w32, col, valid, w[0]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += w[0][i];
                }
            }
            store8(yr + col, valid, y);
        }
    }
}

struct NormBwd {
    const void* dy;         // [N, D]
    const void* x;          // rows, or null with codes
    int64_t ldx;
    const int8_t* codes;
    const uint8_t* scales;
    const float* stats;
    const void* w;
    int w32;
    void* dx;               // [N, D] or null
    float* part;            // [gridDim.x][2][D]: dw, db sums of the block's rows
    int64_t N;
    int D;
};

// Block b walks the rows b·RPB + threadIdx.x / TPR, + gridDim.x·RPB, ...; a
// thread's columns never change, so w and their dw / db sums stay in its
// registers until the end, where the block's row groups add theirs in order.
// The next row is loaded while one is worked on.
template <typename TX, typename TY, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_bwd_kernel(NormBwd a) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    constexpr bool HOLD = NV <= 4;
    __shared__ float part[4][16];
    __shared__ float sums[RPB > 1 ? 2 * TPR * NV * 8 : 1];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int64_t dp = padded(a.D), step = (int64_t)gridDim.x * RPB;
    float dw[NV][8] = {}, db[NV][8] = {};
    float w[HOLD ? NV : 1][8];
    Raw8<TY> gr[NV];
    Raw8<TX> xr[NV];   // or codes in its first half and the scale behind
    float mean_n = 0.0f, rstd_n = 0.0f;
    auto load_row = [&](int64_t row) {
        const float2 st = *reinterpret_cast<const float2*>(a.stats + 2 * row);
        mean_n = st.x, rstd_n = st.y;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j), valid = a.D - col;
            if (valid <= 0) continue;
            gr[j].load(reinterpret_cast<const TY*>(a.dy) + row * a.D + col, valid);
            if (a.codes) {
                const int64_t at = row * dp + col;
                const uint2 c = *reinterpret_cast<const uint2*>(a.codes + at);
                xr[j].q[0] = make_uint4(c.x, c.y, a.scales[at / GROUP], 0u);
            } else {
                xr[j].load(reinterpret_cast<const TX*>(a.x) + row * a.ldx + col, valid);
            }
        }
    };
    int64_t row = (int64_t)blockIdx.x * RPB + grp;
    if constexpr (HOLD) {
        if (row < a.N) load_row(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) load_w<TX>(a.w, a.w32, 8 * (t + TPR * j), a.D - 8 * (t + TPR * j), w[j]);
    }
    int slot = 0;
    for (; row < a.N; row += step) {
        if constexpr (!HOLD) load_row(row);
        const float mean = mean_n, rstd = rstd_n;
        float xh[NV][8], g[NV][8];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (a.D - 8 * (t + TPR * j) <= 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) xh[j][i] = g[j][i] = 0.0f;
                continue;
            }
            gr[j].get(g[j]);
            if (a.codes) decode8(make_uint2(xr[j].q[0].x, xr[j].q[0].y), xr[j].q[0].z, xh[j]);
            else xr[j].get(xh[j]);
        }
        if (HOLD && row + step < a.N) load_row(row + step);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j), valid = a.D - col;
            if (valid <= 0) continue;
            if constexpr (!HOLD) load_w<TX>(a.w, a.w32, col, valid, w[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                xh[j][i] = i < valid ? (xh[j][i] - mean) * rstd : 0.0f;
                dw[j][i] += g[j][i] * xh[j][i];
                db[j][i] += g[j][i];
                g[j][i] *= w[HOLD ? j : 0][i];
                s1 += g[j][i];
                s2 += g[j][i] * xh[j][i];
            }
        }
        if (!a.dx) continue;
        s1 = row_sum<TPR>(s1, part, slot) / (float)a.D;
        s2 = row_sum<TPR>(s2, part, slot + 1) / (float)a.D;
        slot ^= 2;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = 8 * (t + TPR * j), valid = a.D - col;
            if (valid <= 0) continue;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = (g[j][i] - s1 - xh[j][i] * s2) * rstd;
            store8(reinterpret_cast<TX*>(a.dx) + row * a.D + col, valid, o);
        }
    }
    if (!a.part) return;
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.D;
    if constexpr (RPB > 1) {
        // row groups add in order: group 0 writes, each next one adds
        for (int r = 0; r < RPB; ++r) {
            if (grp == r) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float* p = sums + (j * 8 + i) * TPR + t;
                        if (r > 0) {
                            dw[j][i] += p[0];
                            db[j][i] += p[TPR * NV * 8];
                        }
                        if (r < RPB - 1) {
                            p[0] = dw[j][i];
                            p[TPR * NV * 8] = db[j][i];
                        }
                    }
            }
            __syncthreads();
        }
        if (grp != RPB - 1) return;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = 8 * (t + TPR * j), valid = a.D - col;
        if (valid <= 0) continue;
        store8(out + col, valid, dw[j]);
        store8(out + a.D + col, valid, db[j]);
    }
}

// Column sums of part [G][2][D] (G may be 0): dw, and db where given.  A
// block owns 16 columns and splits the G rows over 16 thread rows, each in
// order; the 16 partial sums meet in LDS, in order.
template <typename T>
__global__ __launch_bounds__(256) void col_reduce_kernel(const float* part, int G, int cols, int rowlen, T* out0,
                                                         T* out1, int D) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + c;
    float t = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (int g = r; g < G; g += 16) t += part[(int64_t)g * rowlen + col];
    }
    s[r][c] = t;
    __syncthreads();
    if (r != 0 || col >= cols) return;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += s[i][c];
    if (col < D)
        out0[col] = (T)sum;
    else
        out1[col - D] = (T)sum;
}

// ───────────────────────────── checkpoints ─────────────────────────────

// Rows [N, D] of pitch ldx into codes and scales: a thread per 8-value chunk.
template <typename T>
__global__ __launch_bounds__(256) void pack8_kernel(const T* x, int64_t ldx, int8_t* codes, uint8_t* scales,
                                                    int64_t chunks, int cpr, int D) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= chunks) return;   // whole quads: chunks is a multiple of 4
    const int64_t row = i / cpr;
    const int col = 8 * (int)(i - row * cpr);
    float v[8];
    load8(x + row * ldx + col, D - col, v);
    uint32_t scale;
    const uint2 c = encode8(v, scale);
    *reinterpret_cast<uint2*>(codes + 8 * i) = c;
    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)scale;
}

template <typename T>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t* codes, const uint8_t* scales, T* y,
                                                      int64_t chunks, int cpr, int D) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= chunks) return;
    const int64_t row = i / cpr;
    const int col = 8 * (int)(i - row * cpr);
    float v[8];
    decode8(*reinterpret_cast<const uint2*>(codes + 8 * i), scales[i >> 2], v);
    store8(y + row * D + col, D - col, v);
}

rwkv_status status_of(const char* what) {
    const hipError_t e = hipGetLastError();
    RWKV_REQUIRE(e == hipSuccess, RWKV_E_HIP, "%s: %s", what, hipGetErrorString(e));
    return RWKV_OK;
}

// Blocks of the backward pass: three per CU of 256 threads, two and one of
// more; or one per RPB rows of a small call.  Each writes one partial row of
// dw and db.
int norm_bwd_blocks(int64_t N, int64_t D) {
    const int rpb = D <= 1024 ? 4 : 1, full = D <= 4096 ? 768 : D <= 8192 ? 512 : 256;
    return (int)std::min<int64_t>((N + rpb - 1) / rpb, full);
}

// One wave per row up to 1024 columns, then a block: a thread holds 8 or 16
// values of a row (the backward pass keeps five times as many registers).
#define RWKV_NORM_WIDTHS(RUN)                      \
    if (a.D <= 512) RUN(256, 64, 1)                \
    else if (a.D <= 1024) RUN(256, 64, 2)          \
    else if (a.D <= 2048) RUN(256, 256, 1)         \
    else if (a.D <= 4096) RUN(256, 256, 2)         \
    else if (a.D <= 8192) RUN(512, 512, 2)         \
    else if (a.D <= 16384) RUN(1024, 1024, 2)      \
    else RUN(1024, 1024, 8)

template <typename TX, typename TY>
void norm_fwd_launch(const NormFwd& a, hipStream_t s) {
    // rows beyond a full chip's are walked
    const int64_t blocks = a.D <= 1024 ? (a.N + 3) / 4 : a.N, full = a.D <= 4096 ? 2048 : a.D <= 8192 ? 1024 : 512;
    const dim3 grid((unsigned)std::min(blocks, full));
#define RUN(threads, TPR, NV) rwkv::launch(norm_fwd_kernel<TX, TY, TPR, NV>, grid, dim3(threads), s, a);
    RWKV_NORM_WIDTHS(RUN)
#undef RUN
}

template <typename TX, typename TY>
void norm_bwd_launch(const NormBwd& a, hipStream_t s) {
    const dim3 grid((unsigned)norm_bwd_blocks(a.N, a.D));
#define RUN(threads, TPR, NV) rwkv::launch(norm_bwd_kernel<TX, TY, TPR, NV>, grid, dim3(threads), s, a);
    RWKV_NORM_WIDTHS(RUN)
#undef RUN
}
#undef RWKV_NORM_WIDTHS

// Input and output types a norm takes: the same, or fp32 into 16 bits.
bool norm_types(int x, int y) { return rwkv::dtype_ok(x) && rwkv::dtype_ok(y) && (x == y || x == RWKV_F32); }

}  // namespace

extern "C" {

int64_t rwkv_act8_width(int64_t D) { return D < 1 ? 0 : padded(D); }

rwkv_status rwkv_act8_pack(const void* x, rwkv_dtype dt, int64_t ldx, int8_t* codes, uint8_t* scales, int64_t N,
                           int64_t D, void* stream) {
    RWKV_REQUIRE(rwkv::dtype_ok(dt), RWKV_E_DTYPE, "act8_pack: dtype %d", (int)dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= (1 << 22) && ldx >= D, RWKV_E_SHAPE,
                 "act8_pack: N=%lld D=%lld ldx=%lld", (long long)N, (long long)D, (long long)ldx);
    RWKV_REQUIRE(N == 0 || (x && codes && scales), RWKV_E_NULL, "act8_pack: null buffer");
    if (N == 0) return RWKV_OK;
    const int64_t cpr = padded(D) / 8, chunks = N * cpr, blocks = (chunks + 255) / 256;
    RWKV_REQUIRE(blocks < (int64_t(1) << 31), RWKV_E_SHAPE, "act8_pack: %lld values", (long long)(N * D));
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks);
    if (dt == RWKV_F32)
        rwkv::launch(pack8_kernel<float>, grid, dim3(256), s, (const float*)x, ldx, codes, scales, chunks, (int)cpr, (int)D);
    else if (dt == RWKV_BF16)
        rwkv::launch(pack8_kernel<bf16>, grid, dim3(256), s, (const bf16*)x, ldx, codes, scales, chunks, (int)cpr, (int)D);
    else
        rwkv::launch(pack8_kernel<f16>, grid, dim3(256), s, (const f16*)x, ldx, codes, scales, chunks, (int)cpr, (int)D);
    return status_of("act8_pack launch");
}

rwkv_status rwkv_act8_unpack(const int8_t* codes, const uint8_t* scales, void* y, rwkv_dtype dt, int64_t N, int64_t D,
                             void* stream) {
    RWKV_REQUIRE(rwkv::dtype_ok(dt), RWKV_E_DTYPE, "act8_unpack: dtype %d", (int)dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= (1 << 22), RWKV_E_SHAPE, "act8_unpack: N=%lld D=%lld",
                 (long long)N, (long long)D);
    RWKV_REQUIRE(N == 0 || (codes && scales && y), RWKV_E_NULL, "act8_unpack: null buffer");
    if (N == 0) return RWKV_OK;
    const int64_t cpr = padded(D) / 8, chunks = N * cpr, blocks = (chunks + 255) / 256;
    RWKV_REQUIRE(blocks < (int64_t(1) << 31), RWKV_E_SHAPE, "act8_unpack: %lld values", (long long)(N * D));
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks);
    if (dt == RWKV_F32)
        rwkv::launch(unpack8_kernel<float>, grid, dim3(256), s, codes, scales, (float*)y, chunks, (int)cpr, (int)D);
    else if (dt == RWKV_BF16)
        rwkv::launch(unpack8_kernel<bf16>, grid, dim3(256), s, codes, scales, (bf16*)y, chunks, (int)cpr, (int)D);
    else
        rwkv::launch(unpack8_kernel<f16>, grid, dim3(256), s, codes, scales, (f16*)y, chunks, (int)cpr, (int)D);
    return status_of("act8_unpack launch");
}

rwkv_status rwkv_norm_fwd(const void* x, rwkv_dtype x_dt, int64_t ldx, const void* w, const void* b, rwkv_dtype w_dt,
                          void* y, rwkv_dtype y_dt, float* stats, int8_t* codes, uint8_t* scales, int64_t N, int64_t D,
                          float eps, void* stream) {
    RWKV_REQUIRE(norm_types(x_dt, y_dt) && (w_dt == RWKV_F32 || w_dt == x_dt), RWKV_E_DTYPE,
                 "norm_fwd: types x %d, y %d, weights %d", (int)x_dt, (int)y_dt, (int)w_dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= MAX_D && ldx >= D, RWKV_E_SHAPE,
                 "norm_fwd: N=%lld D=%lld ldx=%lld (D <= %d)", (long long)N, (long long)D, (long long)ldx, MAX_D);
    RWKV_REQUIRE(N == 0 || (x && w && y), RWKV_E_NULL, "norm_fwd: null buffer");
    RWKV_REQUIRE(!codes == !scales, RWKV_E_NULL, "norm_fwd: codes and scales go together");
    if (N == 0) return RWKV_OK;
    const NormFwd a{x, ldx, w, b, w_dt == RWKV_F32, y, stats, codes, scales, N, (int)D, eps};
    const hipStream_t s = (hipStream_t)stream;
    if (x_dt == RWKV_BF16) norm_fwd_launch<bf16, bf16>(a, s);
    else if (x_dt == RWKV_F16) norm_fwd_launch<f16, f16>(a, s);
    else if (y_dt == RWKV_F32) norm_fwd_launch<float, float>(a, s);
    else if (y_dt == RWKV_BF16) norm_fwd_launch<float, bf16>(a, s);
    else norm_fwd_launch<float, f16>(a, s);
    return status_of("norm_fwd launch");
}

int64_t rwkv_norm_bwd_workspace(int64_t N, int64_t D) {
    if (N < 0 || D < 1 || D > MAX_D) return 0;
    return (int64_t)norm_bwd_blocks(N, D) * 2 * D * 4;
}

rwkv_status rwkv_norm_bwd(const void* dy, rwkv_dtype y_dt, const void* x, rwkv_dtype x_dt, int64_t ldx,
                          const int8_t* codes, const uint8_t* scales, const float* stats, const void* w,
                          rwkv_dtype w_dt, void* dx, void* dw, void* db, int64_t N, int64_t D, void* workspace,
                          int64_t workspace_bytes, void* stream) {
    RWKV_REQUIRE(norm_types(x_dt, y_dt) && (w_dt == RWKV_F32 || w_dt == x_dt), RWKV_E_DTYPE,
                 "norm_bwd: types x %d, y %d, weights %d", (int)x_dt, (int)y_dt, (int)w_dt);
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= MAX_D && (codes || ldx >= D), RWKV_E_SHAPE,
                 "norm_bwd: N=%lld D=%lld ldx=%lld (D <= %d)", (long long)N, (long long)D, (long long)ldx, MAX_D);
    RWKV_REQUIRE(!codes == !scales, RWKV_E_NULL, "norm_bwd: codes and scales go together");
    RWKV_REQUIRE(N == 0 || (dy && (x || codes) && stats && w), RWKV_E_NULL, "norm_bwd: null buffer");
    RWKV_REQUIRE(dw || !db, RWKV_E_NULL, "norm_bwd: db without dw");
    const int64_t need = rwkv_norm_bwd_workspace(N, D);
    RWKV_REQUIRE(!dw || need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
                 RWKV_E_SHAPE, "norm_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                 (long long)need);
    const hipStream_t s = (hipStream_t)stream;
    if (N > 0 && (dx || dw)) {
        const NormBwd a{dy, x, ldx, codes, scales, stats, w, w_dt == RWKV_F32, dx, dw ? (float*)workspace : nullptr,
                        N, (int)D};
        if (x_dt == RWKV_BF16) norm_bwd_launch<bf16, bf16>(a, s);
        else if (x_dt == RWKV_F16) norm_bwd_launch<f16, f16>(a, s);
        else if (y_dt == RWKV_F32) norm_bwd_launch<float, float>(a, s);
        else if (y_dt == RWKV_BF16) norm_bwd_launch<float, bf16>(a, s);
        else norm_bwd_launch<float, f16>(a, s);
    }
    if (dw) {
        const int G = norm_bwd_blocks(N, D), cols = (int)(db ? 2 * D : D);
        const dim3 grid((unsigned)((cols + 15) / 16));
        const float* part = (const float*)workspace;
        if (w_dt == RWKV_F32)
            rwkv::launch(col_reduce_kernel<float>, grid, dim3(256), s, part, G, cols, (int)(2 * D), (float*)dw, (float*)db, (int)D);
        else if (w_dt == RWKV_BF16)
            rwkv::launch(col_reduce_kernel<bf16>, grid, dim3(256), s, part, G, cols, (int)(2 * D), (bf16*)dw, (bf16*)db, (int)D);
        else
            rwkv::launch(col_reduce_kernel<f16>, grid, dim3(256), s, part, G, cols, (int)(2 * D), (f16*)dw, (f16*)db, (int)D);
    }
    return status_of("norm_bwd launch");
}

}  // extern "C"
