// Dense products with bias, activation and residual in the epilogue, and
// their gradients, in bf16 and fp16 on the gfx950 matrix cores: the
// projections and low-rank branches of a block in training
// (RWKVBlock.swift:163-307) on dense weights.
//
//   forward   y  = act(x·Wᵀ + b) + res      x [M, K], W [N, K]
//   dz        dz = dy·act'(z), db = Σ_rows dz
//   input     dx = dz·W
//   weight    dW = dzᵀ·x
//
// All three are C[m, n] = Σ_k A[m, k]·B[n, k] over operands that are either
// k-contiguous (x and W of the forward pass, dz of the input gradient) or
// k-major (W of the input gradient, both operands of the weight's), staged in
// LDS as they lie in memory.  k-contiguous rows are read as 16-byte operands;
// k-major ones through ds_read_b64_tr_b16, which hands lane i of sixteen the
// column i of a 4 × 16 block.  Products accumulate in fp32 on
// v_mfma_f32_16x16x32; the epilogue works on the fp32 sums and rounds once.
//
// gemm_dma_kernel (256 × 256, 256 × 128 and 128 × 128 tiles, 16-byte aligned
// rows) is bound by the matrix cores, at the clock that the card holds under
// them (1.7 GHz): 16384 × 14336 × 4096 bf16 in 1.31 ms forward (1470 TFLOP/s),
// 1.33 input gradient, 1.51 weight gradient (whose 896 tiles fill three and a
// half rounds of the 256 CUs).  gemm_kernel (64 × 64 tiles, and rows of any
// alignment) and rows16_kernel take what is bound by latency or W's bytes.
//
// Operand layout of the 16x16x32 instructions (lane l, g = l >> 4, i = l & 15):
// A[m = i][k = 8g .. 8g+7], B[k = 8g .. 8g+7][n = i]; D[m = 4g + r][n = i].

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "act8.h"
#include "launch.h"

namespace {

using namespace rwkv_train;
typedef __bf16 bf16;
typedef _Float16 f16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BK = 64;                   // k per stage: two 32-wide products
constexpr int64_t MAX_LD = RWKV_LINEAR_MAX_PITCH;   // a tile's byte offsets stay under 2^31

template <typename T>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (__is_same(T, bf16))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
}

// ───────────────────────────── epilogue ─────────────────────────────

enum { ACT_NONE = 0, ACT_RELU2 = 1, ACT_TANH = 2, ACT_SIGMOID = 3 };

// What the forward pass keeps for an activation's slope: relu(z), or y for
// bf16 relu², whose root it is; for tanh and sigmoid z, as their values say
// nothing of a slope near zero (1 − h² of a bf16 tanh is 0 from z = 3.5 on).  It
// has 8 bits more than the 16 of its type, which alone would cost more than
// the rounding of dz does.  v and its rounding a
// are neighbours in the order of fp32 bit patterns; the patterns' difference,
// to the nearest of the steps that 8 bits hold, is what a lacks: 16 (bf16) or
// 18 (fp16) bits in all, errors either way.  (128 steps clamp to 127: one value
// in 256 is off by up to a step, the others by half of one, and none comes to
// lie halfway between two values of the type, from where it would go to the
// even one whichever side it was on.)

// Eight values rounded to T (ties to even), packed.
template <typename T>
__device__ __forceinline__ uint4 round8(const float (&v)[8]) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, T2{(T)v[2 * i], (T)v[2 * i + 1]});
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The next 8 bits of the eight values, a what round8 made of them.  (A NaN's
// are any: it stays one.)
template <typename T>
__device__ __forceinline__ uint2 rem8(const float (&v)[8], uint4 a) {
    uint32_t w[8];
    const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]);
        if constexpr (__is_same(T, bf16)) {
            const uint32_t at = i & 1 ? r[i / 2] & 0xffff0000u : r[i / 2] << 16;
            w[i] = (uint32_t)min(max((int)(bits - at + 0x80u) >> 8, -127), 127);
        } else {   // at the type's subnormals the difference is larger: it clamps; an infinity keeps none
            const float f = (float)__builtin_bit_cast(T, (uint16_t)(r[i / 2] >> (16 * (i & 1))));
            const int q = min(max((int)(bits - __builtin_bit_cast(uint32_t, f) + 16u) >> 5, -127), 127);
            w[i] = fabsf(f) <= 65504.0f ? (uint32_t)q : 0u;
        }
    }
    return make_uint2(low_bytes(w[0], w[1], w[2], w[3]), low_bytes(w[4], w[5], w[6], w[7]));
}

template <typename T>
__device__ __forceinline__ float with_rem(float a, uint32_t rem) {
    constexpr int SH = __is_same(T, bf16) ? 8 : 5;
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) + (uint32_t)((int)(int8_t)rem * (1 << SH)));
}

// The first `valid` of eight packed 16-bit values, or bytes.
__device__ __forceinline__ void store_raw(void* p, int valid, uint4 w) {
    if (valid >= 8) {
        __builtin_memcpy(p, &w, 16);
    } else {
#pragma unroll 1
        for (int i = 0; i < valid; ++i) {
            const uint32_t d = i < 4 ? (i < 2 ? w.x : w.y) : (i < 6 ? w.z : w.w);
            reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(d >> (16 * (i & 1)));
        }
    }
}
__device__ __forceinline__ void store_raw(uint8_t* p, int valid, uint2 w) {
    if (valid >= 8) {
        __builtin_memcpy(p, &w, 8);
    } else {
#pragma unroll 1
        for (int i = 0; i < valid; ++i) p[i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

// tanh: the odd Taylor polynomial to x^11 where |x| < 0.35 (the next term is
// under 2^-26 of x), else (1 − t)/(1 + t), t = e^(−2|x|).
__device__ __forceinline__ float tanh_of(float x) {
    const float s = x * x;
    const float p = x * (1.0f + s * (-1.0f / 3 + s * (2.0f / 15 + s * (-17.0f / 315 + s * (62.0f / 2835 + s * (-1382.0f / 155925))))));
    const float t = __builtin_amdgcn_exp2f(fabsf(x) * -2.885390081777927f);
    const float q = __builtin_copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
    return fabsf(x) < 0.35f ? p : q;
}

__device__ __forceinline__ float sigmoid_of(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

// Slopes by t = e^(−2|z|) and e^(−|z|), as precise near zero as elsewhere:
// 1 − tanh² = 4t/(1 + t)², σ(1 − σ) = t/(1 + t)².
__device__ __forceinline__ float tanh_slope(float z) {
    const float t = __builtin_amdgcn_exp2f(fabsf(z) * -2.885390081777927f), r = __builtin_amdgcn_rcpf(1.0f + t);
    return 4.0f * t * r * r;
}

__device__ __forceinline__ float sigmoid_slope(float z) {
    const float t = __builtin_amdgcn_exp2f(fabsf(z) * -1.4426950408889634f), r = __builtin_amdgcn_rcpf(1.0f + t);
    return t * r * r;
}

struct Epilogue {
    const void* bias;     // [N] of the operands' type, or null
    const void* res;      // [M] rows of pitch ldr, or null
    int64_t ldr;
    void* y;              // [M, N]
    int wide;             // res and y are fp32 (else the operands' type)
    void* aux;            // [M, N] of the operands' type: relu(z) with relu², else z; or null
    uint8_t* rem;         // [M, N]: the next 8 bits of aux, without aux of relu²'s y; or null
    int8_t* codes;        // checkpoint of z, [M, Np]; or null
    uint8_t* scales;
    int act;
    int64_t M;
    int N;
    bool plain;           // y alone, of the operands' type
};

// Eight neighbouring columns of each of C rows row, row + step, ..., z without
// bias in v.  Every flag is looked at once for all of them.  With codes, the
// four lanes of a 32-column group call it together.
template <typename T, int C>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t row, int step, int col, float (&v)[C][8]) {
    const int valid = e.N - col;
    if (e.bias) {
        float b[8];
        load8(reinterpret_cast<const T*>(e.bias) + col, valid, b);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] += b[i];
    }
    if (e.codes) {
        const int64_t np = padded(e.N);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (valid < 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = i < valid ? v[c][i] : 0.0f;
            }
            uint32_t scale;
            const uint2 code = encode8(v[c], scale);
            if (col < np && row + c * step < e.M) {
                const int64_t at = (row + c * step) * np + col;
                *reinterpret_cast<uint2*>(e.codes + at) = code;
                if ((col & 31) == 0) e.scales[at / GROUP] = (uint8_t)scale;
            }
        }
    }
    const int64_t at = row * e.N + col, pitch = (int64_t)step * e.N;
    if (e.act == ACT_RELU2) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] < 0.0f ? 0.0f : v[c][i];   // a NaN stays one
    }
    if (e.aux) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (row + c * step < e.M) {
                const uint4 a = round8<T>(v[c]);
                store_raw(reinterpret_cast<T*>(e.aux) + at + c * pitch, valid, a);
                store_raw(e.rem + at + c * pitch, valid, rem8<T>(v[c], a));
            }
    }
    if (e.act == ACT_RELU2) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] *= v[c][i];
    } else if (e.act == ACT_TANH) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = tanh_of(v[c][i]);
    } else if (e.act == ACT_SIGMOID) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = sigmoid_of(v[c][i]);
    }
    if (e.rem && !e.aux) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (row + c * step < e.M) store_raw(e.rem + at + c * pitch, valid, rem8<T>(v[c], round8<T>(v[c])));
    }
    if (e.res) {
        float s[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t from = min(row + c * step, e.M - 1) * e.ldr + col;   // all C loads before their use
            if (e.wide)
                load8(reinterpret_cast<const float*>(e.res) + from, valid, s[c]);
            else
                load8(reinterpret_cast<const T*>(e.res) + from, valid, s[c]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] += s[c][i];
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (row + c * step >= e.M) continue;
        if (e.wide)
            store8(reinterpret_cast<float*>(e.y) + at + c * pitch, valid, v[c]);
        else
            store_raw(reinterpret_cast<T*>(e.y) + at + c * pitch, valid, round8<T>(v[c]));
    }
}

// ───────────────────────────── operand tiles ─────────────────────────────

// ROWS output rows (or columns) × BK of an operand: how a workgroup loads a
// stage of it into registers, writes it to LDS and reads operands back.  ODD:
// rows that are not 16-byte aligned or a k-contiguous length that 8 does not
// divide; elsewhere buffer loads, whose range check fills what lies outside
// the operand with zeros.
template <typename T, bool KM, int ROWS, int THREADS, bool ODD>
struct Tile {
    static constexpr int P = ROWS * 8 / THREADS;   // 16-byte chunks per thread and stage
    static constexpr int CPR = KM ? ROWS / 8 : 8;  // chunks per LDS row
    static constexpr int STEP = THREADS / CPR;     // LDS rows a thread's chunks are apart
    static constexpr int BYTES = ROWS * BK * 2;
    static_assert(P >= 1 && THREADS % CPR == 0, "tile shape");

    const T* p;       // operand, at the tile's first row (k-contiguous) or column (k-major)
    int64_t ld;
    int rows;         // rows (columns) from there to the operand's end
    int K;
    int c, r;         // the thread's chunk and first LDS row
    bool whole;       // the operand's rows hold a chunk

    __device__ __forceinline__ Tile(const void* base, int64_t ld_, int64_t at, int64_t total, int K_, int tid)
        : p(reinterpret_cast<const T*>(base) + (KM ? at : at * ld_)), ld(ld_),
          rows((int)min(total - at, (int64_t)(KM ? (1 << 30) : ROWS))), K(K_), c(tid % CPR), r(tid / CPR),
          whole((KM ? total : (int64_t)K_) >= 8) {}

    __device__ __forceinline__ void load(uint4 (&v)[P], int st) const {
        if constexpr (ODD) {
            // A chunk that would pass the row's end is loaded as the row's last
            // whole one (fix() moves its values): every load is unconditional
            // and none is looked at before it is written to LDS.
            if (whole) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int row = r + STEP * i;
                    const T* q = p + (KM ? (int64_t)min(st * BK + row, K - 1) * ld : (int64_t)min(row, rows - 1) * ld) + from(st);
                    __builtin_memcpy(&v[i], q, 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int row = r + STEP * i;
                    const int k = KM ? st * BK + row : st * BK + 8 * c;
                    const int valid = KM ? (k < K ? rows - 8 * c : 0) : (row < rows ? K - k : 0);
                    const T* q = p + (KM ? (int64_t)k * ld + 8 * c : (int64_t)row * ld + k);
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 7; ++e)
                        if (e < valid) w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[e] << (16 * (e & 1));
                    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        } else if constexpr (KM) {
            const int left = min(BK, K - st * BK);   // rows of this stage
            // whole dwords: one that holds a last odd column may be read
            const int cols = (min(rows, ROWS) + 1) & ~1;
            const int bytes = left > 0 ? (int)(((int64_t)(left - 1) * ld + cols) * 2) : 0;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(p + (left > 0 ? (int64_t)st * BK * ld : 0)), 0, bytes, 0x00020000);
            const uint32_t o = (uint32_t)(r * (int)ld + 8 * c) * 2, step = (uint32_t)(STEP * (int)ld) * 2;
#pragma unroll
            for (int i = 0; i < P; ++i)
                v[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, o + i * step, 0, 0));
        } else {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(p), 0, (int)(((int64_t)(rows - 1) * ld + K) * 2), 0x00020000);
            const int k = st * BK + 8 * c;
            // past the last k: an offset outside the range (also after the row steps are added)
            const uint32_t o = k < K ? (uint32_t)(r * (int)ld + k) * 2 : 0x80000000u;
            const uint32_t step = (uint32_t)(STEP * (int)ld) * 2;
#pragma unroll
            for (int i = 0; i < P; ++i)
                v[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, o + i * step, 0, 0));
        }
    }

    // Column (of a k-major row, or k) at which the thread's chunk is loaded.
    __device__ __forceinline__ int from(int st) const { return KM ? min(8 * c, rows - 8) : min(st * BK + 8 * c, K - 8); }

    // Stage st's chunks as loaded into what they stand for: zeros past the end.
    __device__ __forceinline__ void fix(uint4 (&v)[P], int st) const {
        if constexpr (!ODD) return;
        const bool tail = (st + 1) * BK > K;
        if (!whole || !(tail || (KM && rows < ROWS))) return;
        const int moved = (KM ? 8 * c : st * BK + 8 * c) - from(st);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            uint64_t lo = (uint64_t)v[i].y << 32 | v[i].x, hi = (uint64_t)v[i].w << 32 | v[i].z;
            if (moved >= 4) lo = hi, hi = 0;
            const int sh = 16 * (moved & 3);
            lo = lo >> sh | (hi << 1) << (63 - sh);
            hi >>= sh;
            if (moved >= 8 || (KM && st * BK + r + STEP * i >= K)) lo = hi = 0;
            v[i] = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
        }
    }

    // 32-byte slots of a k-major LDS row are permuted by the row, so that the
    // eight rows a half wave reads at once lie in different banks (rows of
    // 128 bytes: two rows share the banks' width).
    static __device__ __forceinline__ int slot_mask(int k) {
        return ROWS >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
    }

    __device__ __forceinline__ void write(char* lds, const uint4 (&v)[P]) const {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int row = r + STEP * i;
            const int at = KM ? row * ROWS * 2 + (((c >> 1) ^ slot_mask(row)) << 5) + ((c & 1) << 4)
                              : row * 128 + ((c ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(lds + at) = v[i];
        }
    }

    // The operand of rows base + 16·tile + i (i = lane & 15), k = 32·kk + 8g ..
    // 8g + 7; base a multiple of 16.
    static __device__ __forceinline__ uint4 frag(char* lds, int base, int tile, int kk, int lane) {
        const int g = lane >> 4, i = lane & 15;
        if constexpr (KM) {
            typedef __attribute__((address_space(3))) s16x4* lptr;
            const int k = 32 * kk + 8 * g + (i >> 2);
            const int s = slot_mask(k);   // the same for k + 4 (bit 2 takes no part)
            const int col = (((base >> 4) + tile) ^ s) * 32 + (i & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(lds + k * ROWS * 2 + col));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(lds + (k + 4) * ROWS * 2 + col));
            const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(uint4, v);
        } else {
            const int row = base + 16 * tile + i;
            return *reinterpret_cast<const uint4*>(lds + row * 128 + (((4 * kk + g) ^ (row & 7)) << 4));
        }
    }
};

struct GemmArgs {
    const void* a;
    int64_t lda;          // k-contiguous: [M][lda]; k-major: [K][lda]
    const void* b;
    int64_t ldb;
    int64_t M;
    int N, K;
    int KB;               // rows of a k-major B: K, or less where A's last columns are padding zeros
    int full;             // tiles taken whole; the others in `splits` K ranges of `per` stages each,
    int splits, per;      //   fp32 sums into part [splits][tiles - full][tile]
    float* part;
    Epilogue e;
};

// Tile `id`: tiles in groups of 4 row blocks × every column
// block, column-major within a group; XCD x (workgroups x, x + 8, ...) takes a
// contiguous run of that order, so its workgroups share operand blocks in its
// L2.
__device__ __forceinline__ void tile_of(int id, int ntm, int ntn, int& tm, int& tn) {
    const int total = ntm * ntn, xcd = id & 7, loc = id >> 3;
    const int t = xcd * (total >> 3) + min(xcd, total & 7) + loc;
    const int grp = t / (4 * ntn), first = 4 * grp, gm = min(4, ntm - first);
    const int rr = t - grp * 4 * ntn;
    tm = first + rr % gm;
    tn = rr / gm;
}

// A workgroup's piece: a tile, and the stages of it.
struct Item {
    int tm, tn, st0, st1;
    int part;   // index of its partial tile; -1: the tile is whole
};
__device__ __forceinline__ Item item_of(const GemmArgs& g, int id, int ntm, int ntn) {
    const int rest = ntm * ntn - g.full, nst = (g.K + BK - 1) / BK;
    Item it;
    if (id < g.full) {
        tile_of(id, ntm, ntn, it.tm, it.tn);
        it.st0 = 0, it.st1 = nst, it.part = -1;
    } else {
        it.part = id - g.full;
        const int split = it.part / rest;
        tile_of(g.full + it.part - split * rest, ntm, ntn, it.tm, it.tn);
        it.st0 = split * g.per, it.st1 = min(nst, it.st0 + g.per);
    }
    return it;
}
__device__ __forceinline__ int items_of(const GemmArgs& g, int ntm, int ntn) {
    return g.full + (ntm * ntn - g.full) * g.splits;
}

// A wave's 16·AM × 16·AN products, RC row tiles at a time through its own
// 16·RC · EROW floats of LDS, so that a lane gets eight neighbouring columns;
// or into the wave's place in a partial tile, if there is one.
template <int AN>
constexpr int EROW = 16 * AN + 4;   // floats per staged row

template <typename T, int AM, int AN, int RC>
__device__ __forceinline__ void finish_tile(const GemmArgs& g, const f32x4 (&acc)[AM][AN], float* stage, int64_t row0,
                                            int col0, int lane, float* part, int pitch) {
    static_assert(AM % RC == 0, "row tiles per pass");
    constexpr int LPR = 2 * AN, RPP = 64 / LPR;   // lanes per row, rows per step
    const int gq = lane >> 4, li = lane & 15;
    const int cl = 8 * (lane % LPR), col = col0 + cl;
#pragma unroll
    for (int h = 0; h < AM / RC; ++h) {
#pragma unroll
        for (int i = 0; i < RC; ++i)
#pragma unroll
            for (int j = 0; j < AN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    stage[(16 * i + 4 * gq + q) * EROW<AN> + 16 * j + li] = acc[h * RC + i][j][q];
        __builtin_amdgcn_wave_barrier();
        constexpr int C = 16 * RC / RPP < 4 ? 16 * RC / RPP : 4;   // rows of a lane per round
#pragma unroll 1
        for (int rloc = lane / LPR; rloc < 16 * RC; rloc += C * RPP) {
            const int64_t row = row0 + h * 16 * RC + rloc;
            float v[C][8];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float4 lo = *reinterpret_cast<const float4*>(stage + (rloc + c * RPP) * EROW<AN> + cl);
                const float4 hi = *reinterpret_cast<const float4*>(stage + (rloc + c * RPP) * EROW<AN> + cl + 4);
                v[c][0] = lo.x; v[c][1] = lo.y; v[c][2] = lo.z; v[c][3] = lo.w;
                v[c][4] = hi.x; v[c][5] = hi.y; v[c][6] = hi.z; v[c][7] = hi.w;
            }
            if (part) {
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (row + c * RPP < g.M) store8(part + (h * 16 * RC + rloc + c * RPP) * pitch + cl, 8, v[c]);
            } else {
                finish<T, C>(g.e, row, RPP, col, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, bool AKM, bool BKM, int WM, int WN, int AM, int AN, bool ODD>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs g) {
    constexpr int BM = 16 * WM * AM, BN = 16 * WN * AN, THREADS = 64 * WM * WN;
    using TileA = Tile<T, AKM, BM, THREADS, ODD>;
    using TileB = Tile<T, BKM, BN, THREADS, ODD>;
    constexpr int STAGE = TileA::BYTES + TileB::BYTES;
    static_assert(WM * WN * 32 * EROW<AN> * 4 <= 2 * STAGE, "epilogue staging");
    __shared__ __align__(16) char lds[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ntm = (int)((g.M + BM - 1) / BM), ntn = (g.N + BN - 1) / BN, tiles = ntm * ntn;
    const Item it = item_of(g, blockIdx.x, ntm, ntn);
    const int64_t m0 = (int64_t)it.tm * BM;
    const int n0 = it.tn * BN;
    const int st0 = it.st0, st1 = it.st1;

    const TileA ta(g.a, g.lda, m0, g.M, g.K, tid);
    const TileB tb(g.b, g.ldb, n0, g.N, g.KB, tid);
    const int wm = wave % WM, wn = wave / WM;
    f32x4 acc[AM][AN];
#pragma unroll
    for (int i = 0; i < AM; ++i)
#pragma unroll
        for (int j = 0; j < AN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    uint4 va[TileA::P], vb[TileB::P];
    ta.load(va, st0);
    tb.load(vb, st0);
    ta.fix(va, st0);
    tb.fix(vb, st0);
    ta.write(lds, va);
    tb.write(lds + TileA::BYTES, vb);
    ta.load(va, st0 + 1);
    tb.load(vb, st0 + 1);
    __syncthreads();
    for (int st = st0; st < st1; ++st) {
        char* cur = lds + ((st - st0) & 1) * STAGE;
        char* nxt = lds + ((st - st0 + 1) & 1) * STAGE;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint4 av[AM], bv[AN];
#pragma unroll
            for (int j = 0; j < AN; ++j) bv[j] = TileB::frag(cur + TileA::BYTES, wn * AN * 16, j, kk, lane);
#pragma unroll
            for (int i = 0; i < AM; ++i) av[i] = TileA::frag(cur, wm * AM * 16, i, kk, lane);
            if (kk == 1) {   // the next stage's chunks, then the loads of the one after
                ta.fix(va, st + 1);
                tb.fix(vb, st + 1);
                ta.write(nxt, va);
                tb.write(nxt + TileA::BYTES, vb);
                ta.load(va, st + 2);
                tb.load(vb, st + 2);
            }
#pragma unroll
            for (int i = 0; i < AM; ++i)
#pragma unroll
                for (int j = 0; j < AN; ++j) acc[i][j] = mfma<T>(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }

    float* const part = it.part < 0 ? nullptr : g.part + (int64_t)it.part * BM * BN + wm * AM * 16 * BN + wn * AN * 16;
    finish_tile<T, AM, AN, 2>(g, acc, reinterpret_cast<float*>(lds) + wave * 32 * EROW<AN>, m0 + wm * AM * 16,
                              n0 + wn * AN * 16, lane, part, BN);
}

// ───────────────────────────── whole tiles: loads straight into LDS ─────────────────────────────

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes per lane from a buffer into LDS at m0 + 16·lane (bytes).  The
// compiler does not know of these loads: whoever reads the LDS bytes waits for
// vmcnt first.  Offsets outside the buffer store zeros.  m0 is set a product
// earlier (an instruction has to lie between); nothing else here uses it.
template <int ADD>
__device__ __forceinline__ void lds_target(uint32_t at) {
    asm volatile("s_add_u32 m0, %0, %1" ::"s"(at), "n"(ADD) : "scc");
}
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t off) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc));
}

template <typename F, int... I>
__device__ __forceinline__ void unrolled(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

__device__ __forceinline__ i32x4 rsrc_of(uint64_t base, uint32_t bytes) {
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)base), __builtin_amdgcn_readfirstlane((int)(base >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

// ROWS × BK of an operand with 16-byte aligned rows, as Tile lays it out.  A
// load covers 1024 LDS bytes; the permutation of the LDS layout is applied to
// the global addresses its lanes read.
template <typename T, bool KM, int ROWS, int WAVES, bool FEW>
struct DmaTile {
    static constexpr int P = ROWS / 8 / WAVES;       // loads per wave and stage
    static constexpr int KR = KM ? 512 / ROWS : 0;   // k rows per load
    static constexpr int BYTES = ROWS * BK * 2;
    static_assert(P >= 1, "tile shape");
    using Read = Tile<T, KM, ROWS, 64 * WAVES, false>;

    i32x4 r;           // the stage's part of the tile
    int64_t ld;
    int k, cols;       // k from the stage's start to the operand's end; k-major: columns, to whole dwords
    uint32_t x;        // k-contiguous: sends offsets past the last k out of range
    // the lane's byte offset of each load; FEW: of the first, odd and even, where
    // registers are short (k-major)
    uint32_t off[FEW && KM ? 2 : P];
    int c;             // k-contiguous: the lane's k within a stage

    __device__ __forceinline__ DmaTile(int64_t ld_, int wave, int lane) : r{}, ld(ld_), k(0), cols(0), x(0), c(0) {
#pragma unroll
        for (int j = 0; j < P; ++j) {   // LDS bytes 1024·(j·WAVES + wave) of the tile
            if constexpr (KM) {
                if (FEW && j > 1) continue;
                const int kr = (j * WAVES + wave) * KR + lane / (ROWS / 8), pos = lane % (ROWS / 8);
                const int chunk = (((pos >> 1) ^ Read::slot_mask(kr)) << 1) | (pos & 1);
                off[j] = (uint32_t)(kr * (int)ld + 8 * chunk) * 2;
            } else {
                const int row = (j * WAVES + wave) * 8 + (lane >> 3);
                c = 8 * ((lane & 7) ^ (row & 7));   // the same for every j
                off[j] = (uint32_t)(row * (int)ld + c) * 2;
            }
        }
    }
    template <int j>
    __device__ __forceinline__ uint32_t at() const {
        if constexpr (FEW && KM) return off[j & 1] + (uint32_t)((j >> 1) * 2 * WAVES * KR * (int)ld) * 2;
        else return KM ? off[j] : off[j] | x;
    }

    // Row (column) `at` of `total`, stage st of an operand of K.
    __device__ __forceinline__ void start(const void* base, int64_t at, int64_t total, int K, int st) {
        const int rows = (int)min(total - at, (int64_t)ROWS);
        k = K - st * BK;
        // a dword that holds a last odd column may be read whole
        cols = (rows + 1) & ~1;
        const uint64_t p = (uint64_t)base + (KM ? (uint64_t)at + (uint64_t)st * BK * (uint64_t)ld : (uint64_t)at * ld + (uint64_t)st * BK) * 2;
        r = rsrc_of(p, k <= 0 ? 0u : KM ? bytes() : (uint32_t)(((int64_t)(rows - 1) * ld + k) * 2));
        x = beyond();
    }
    __device__ __forceinline__ void end() { k = 0, r[2] = 0; }   // loads out of range from here on

    // To the next stage, in steps that fit between products.
    __device__ __forceinline__ void next_base() {
        const uint64_t p = ((uint64_t)(uint32_t)r[1] << 32 | (uint32_t)r[0]) + (KM ? (uint64_t)BK * (uint64_t)ld * 2 : BK * 2);
        r[0] = (int)(uint32_t)p;
        r[1] = (int)(p >> 32);
        k -= BK;
    }
    __device__ __forceinline__ void next_bytes() {
        if constexpr (KM) r[2] = k >= BK ? r[2] : k > 0 ? (int)bytes() : 0;
        else r[2] = k > 0 ? r[2] - BK * 2 : 0;
    }
    __device__ __forceinline__ void next_beyond() { x = beyond(); }

private:
    __device__ __forceinline__ uint32_t bytes() const { return (uint32_t)(((int64_t)(min(k, BK) - 1) * ld + cols) * 2); }
    __device__ __forceinline__ uint32_t beyond() const { return KM || c < k ? 0u : 0x80000000u; }
};

enum { EPI_PLAIN, EPI_PART, EPI_FULL };

// C = A·Bᵀ.  A workgroup walks the items (tile, K range) blockIdx.x,
// + gridDim.x, ...; its loads run two stages ahead of the products
// straight through the items' ends.  A stage is two halves of 32 k: while the
// matrix cores work on one half's operands the other's are read.  After two
// thirds of the first half every wave has read the stage's buffer, which is
// refilled from there on; at three eighths of the second half the next stage's
// loads have to be done.  One wave per SIMD issues everything, so whatever is
// not a product stands between products a few instructions at a time: the
// loader's step to the next stage in one piece cost 8 % of the kernel.
//
// The products are taken as (B tile)·(A tile)ᵀ, so that a lane holds four
// neighbouring columns of a row: columns 16j + 4g .. + 3 of row 16i + (l & 15).
template <typename T, bool AKM, bool BKM, int WM, int WN, int AM, int AN, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 1) void gemm_dma_kernel(GemmArgs g) {
    constexpr int BM = 16 * WM * AM, BN = 16 * WN * AN, W = WM * WN;
    using DA = DmaTile<T, AKM, BM, W, EPI == EPI_PART>;
    using DB = DmaTile<T, BKM, BN, W, EPI == EPI_PART>;
    using TileA = typename DA::Read;
    using TileB = typename DB::Read;
    constexpr uint32_t STAGE = DA::BYTES + DB::BYTES;
    constexpr int NM = AM * AN, NF = AM + AN, ND = DA::P + DB::P;
    // Within a stage's 2·NM products: operands are read beside every RM-th
    // product from the half's start (from MB in the second half), loads are
    // issued beside every LM-th from MA in the first half on, spread as far as
    // they go: the texture path takes 64 bytes a cycle, half of a stage's time.
    constexpr int RM = NM / 2 / NF, MA = NM * 11 / 16, MB = NM * 3 / 8, LM = (2 * NM - MA) / ND;
    static_assert(RM * NF <= MA && MB + RM * NF <= NM && MA + LM * ND <= 2 * NM, "places of a stage");
    constexpr int SM = MA / 6;   // the loader's steps: beside every SM-th before MA
    constexpr int CPR = 4 * AN;   // 16-byte chunks of a staged row of the epilogue
    __shared__ __align__(1024) char lds[2 * STAGE + (EPI == EPI_PART ? 0 : W * 16 * CPR * 16)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ntm = (int)((g.M + BM - 1) / BM), ntn = (g.N + BN - 1) / BN;
    // the whole tiles, or the pieces of the others
    const int first = (EPI == EPI_PART ? g.full : 0) + blockIdx.x, items = EPI == EPI_PART ? items_of(g, ntm, ntn) : g.full;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const int wm = wave % WM, wn = wave / WM;

    // the loader: its item, the stages left of it, and the operands' parts of
    // its stage; a step to the next stage has six parts
    DA da(g.lda, wave, lane);
    DB db(g.ldb, wave, lane);
    int l_item = first, l_left = 0;
    auto start = [&] {
        if (l_item < items) {
            const Item it = item_of(g, l_item, ntm, ntn);
            da.start(g.a, (int64_t)it.tm * BM, g.M, g.K, it.st0);
            db.start(g.b, (int64_t)it.tn * BN, g.N, g.KB, it.st0);
            l_left = it.st1 - it.st0;
        } else {
            da.end();
            db.end();
            l_left = 1 << 30;
        }
    };
    auto step = [&](auto part) {
        if constexpr (part == 0) da.next_base();
        if constexpr (part == 1) da.next_bytes();
        if constexpr (part == 2) db.next_base();
        if constexpr (part == 3) db.next_bytes();
        if constexpr (part == 4) da.next_beyond(), db.next_beyond();
        if constexpr (part == 5)
            if (--l_left == 0) {
                l_item += gridDim.x;
                start();
            }
    };
    // load j of a wave into its buffer: target and load
    auto target = [&](uint32_t buf, auto j) {
        lds_target<(j < DA::P ? 0 : DA::BYTES) + (j < DA::P ? j : j - DA::P) * W * 1024>(base + buf + wave * 1024);
    };
    auto load = [&](auto j) {
        if constexpr (j < DA::P) load_to_lds(da.r, da.template at<j>());
        else load_to_lds(db.r, db.template at<j - DA::P>());
    };
    auto load_all = [&](uint32_t buf) {
        unrolled([&](auto j) {
            target(buf, j);
            asm volatile("s_nop 0");
            load(j);
        }, std::make_integer_sequence<int, ND>{});
    };

    f32x4 acc[AM][AN];
    uint4 av[2][AM], bv[2][AN];
    auto read = [&](int set, int kk, uint32_t buf, int f) {
        if (f < AN) bv[set][f] = TileB::frag(lds + buf + DA::BYTES, wn * AN * 16, f, kk, lane);
        else av[set][f - AN] = TileA::frag(lds + buf, wm * AM * 16, f - AN, kk, lane);
    };
    start();
    load_all(0);
    unrolled(step, std::make_integer_sequence<int, 6>{});
    load_all(STAGE);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ND) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int f = 0; f < NF; ++f) read(0, 0, 0, f);
    uint32_t cur = 0;
    for (int item = first; item < items; item += gridDim.x) {
        const Item it = item_of(g, item, ntm, ntn);
        const int count = it.st1 - it.st0;
#pragma unroll
        for (int i = 0; i < AM; ++i)
#pragma unroll
            for (int j = 0; j < AN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int st = 0; st < count; ++st) {
            unrolled([&](auto m) {
                if constexpr (m == MA) {   // every wave has read this stage's buffer
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                if constexpr (m % SM == SM - 1 && m / SM < 6) step(std::integral_constant<int, m / SM>{});
                constexpr bool dma = m >= MA && (m - MA) % LM == 0 && (m - MA) / LM < ND;
                if constexpr (dma) {
                    target(cur, std::integral_constant<int, (m - MA) / LM>{});
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (m % RM == 0 && m / RM < NF) read(1, 1, cur, m / RM);
                acc[m / AN][m % AN] = mfma<T>(bv[0][m % AN], av[0][m / AN], acc[m / AN][m % AN]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (dma) load(std::integral_constant<int, (m - MA) / LM>{});
                __builtin_amdgcn_sched_barrier(0);
            }, std::make_integer_sequence<int, NM>{});
            unrolled([&](auto m) {
                constexpr int at = NM + m - MA;   // loads' place
                if constexpr (m == MB) {   // the next stage's loads are done in every wave
                    constexpr int issued = (at + LM - 1) / LM < ND ? (at + LM - 1) / LM : ND;
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(issued) : "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                constexpr bool dma = at % LM == 0 && at / LM < ND;
                if constexpr (dma) {
                    target(cur, std::integral_constant<int, at / LM>{});
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (m >= MB && (m - MB) % RM == 0 && (m - MB) / RM < NF) read(0, 0, cur ^ STAGE, (m - MB) / RM);
                acc[m / AN][m % AN] = mfma<T>(bv[1][m % AN], av[1][m / AN], acc[m / AN][m % AN]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (dma) load(std::integral_constant<int, at / LM>{});
                __builtin_amdgcn_sched_barrier(0);
            }, std::make_integer_sequence<int, NM>{});
            cur ^= STAGE;
        }

        int l = lane;
        asm volatile("" : "+v"(l));   // addresses are formed here, not kept over the products
        const int64_t row0 = (int64_t)it.tm * BM + wm * AM * 16;
        const int col0 = it.tn * BN + wn * AN * 16, gq = l >> 4, li = l & 15;
        if constexpr (EPI == EPI_PART) {
            float* p = g.part + (int64_t)it.part * BM * BN + (wm * AM * 16 + li) * BN + wn * AN * 16 + 4 * gq;
            int left = (int)min(g.M - row0, (int64_t)BM) - li;   // rows from the lane's on
#pragma unroll
            for (int i = 0; i < AM; ++i, left -= 16, p += 16 * BN) {
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" : "+v"(p), "+v"(left));   // stepped, not formed ahead
                if (left <= 0) continue;
#pragma unroll
                for (int j = 0; j < AN; ++j) *reinterpret_cast<f32x4*>(p + 16 * j) = acc[i][j];
            }
        } else {
            // sixteen rows at a time through LDS of the wave's own; a rolled
            // loop, as the finishing code is long
            float4* const own = reinterpret_cast<float4*>(lds + 2 * STAGE) + wave * 16 * CPR;
#pragma unroll 1
            for (int i = 0; i < AM; ++i) {
#pragma unroll
                for (int k = 0; k < AM; ++k) {
                    if (i != k) continue;
#pragma unroll
                    for (int j = 0; j < AN; ++j)
                        own[li * CPR + ((4 * j + gq) ^ li)] = make_float4(acc[k][j][0], acc[k][j][1], acc[k][j][2], acc[k][j][3]);
                }
                __builtin_amdgcn_wave_barrier();
                constexpr int LPR = CPR / 2, RPP = 64 / LPR, C = 16 / RPP;   // lanes per row, rows per step
                const int q = l % LPR;
                float v[C][8];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int r = c * RPP + l / LPR;
                    const float4 lo = own[r * CPR + ((2 * q) ^ r)], hi = own[r * CPR + ((2 * q + 1) ^ r)];
                    v[c][0] = lo.x; v[c][1] = lo.y; v[c][2] = lo.z; v[c][3] = lo.w;
                    v[c][4] = hi.x; v[c][5] = hi.y; v[c][6] = hi.z; v[c][7] = hi.w;
                }
                const int64_t row = row0 + 16 * i + l / LPR;
                const int col = col0 + 8 * q;
                if constexpr (EPI == EPI_FULL) {
                    finish<T, C>(g.e, row, RPP, col, v);
                } else {
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        if (row + c * RPP < g.M)
                            store_raw(reinterpret_cast<T*>(g.e.y) + (row + c * RPP) * g.N + col, g.N - col, round8<T>(v[c]));
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // loads of stages that do not come still write LDS
}

// Sums the K ranges of the tiles from g.full on, in order, and finishes them:
// a thread per 8 columns.
template <typename T>
__global__ __launch_bounds__(256) void split_reduce_kernel(GemmArgs g, int BM, int BN, int ntm, int ntn) {
    const int rest = ntm * ntn - g.full, per = BM * BN / 8 / 256;   // blocks per tile
    const int t = blockIdx.x / per, at = (blockIdx.x - t * per) * 256 + threadIdx.x;
    int tm, tn;
    tile_of(g.full + t, ntm, ntn, tm, tn);
    const int r = at / (BN / 8), c = 8 * (at - r * (BN / 8));
    const int64_t row = (int64_t)tm * BM + r;
    if (row >= g.M) return;   // whole quads: a row's chunks
    const int col = tn * BN + c;
    const float* p = g.part + ((int64_t)t * BM + r) * BN + c;
    float v[1][8] = {};
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
        float q[8];
        load8(p + (int64_t)s * rest * BM * BN, 8, q);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[0][k] += q[k];
    }
    finish<T, 1>(g.e, row, 1, col, v);
}

// ───────────────────────────── a few rows ─────────────────────────────

// x [M <= 16, K] through W: a block takes 16·NT columns (rows of W), its eight
// waves every eighth 32 of k, straight from memory into the products' operands
// (any alignment), the next U of each on their way under U products; their
// sums meet in LDS, in order.
template <typename T, int NT>
__global__ __launch_bounds__(512) void rows16_kernel(GemmArgs g) {
    constexpr int WAVES = 8, U = 8 / NT;
    __shared__ __align__(16) float sums[WAVES][16][16 * NT + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
    const int n0 = blockIdx.x * 16 * NT, steps = (g.K + 31) / 32;
    const T* xr = reinterpret_cast<const T*>(g.a) + (int64_t)min(i, (int)g.M - 1) * g.lda;
    const T* wr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wr[t] = reinterpret_cast<const T*>(g.b) + (int64_t)min(n0 + 16 * t + i, g.N - 1) * g.ldb;
    auto chunk = [&](const T* p, int k) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (k + 8 <= g.K) {
            __builtin_memcpy(&v, p + k, 16);
        } else if (k < g.K) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
            for (int e = 0; e < 7; ++e)
                if (k + e < g.K) w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[k + e] << (16 * (e & 1));
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return v;
    };
    uint4 w[NT][U], x[U];
    auto load = [&](int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s + WAVES * u) * 32 + 8 * q;
            x[u] = chunk(xr, k);
#pragma unroll
            for (int t = 0; t < NT; ++t) w[t][u] = chunk(wr[t], k);
        }
    };
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    load(wave);
    for (int s = wave; s < steps; s += WAVES * U) {
        uint4 cw[NT][U], cx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            cx[u] = x[u];
#pragma unroll
            for (int t = 0; t < NT; ++t) cw[t][u] = w[t][u];
        }
        if (s + WAVES * U < steps) load(s + WAVES * U);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = mfma<T>(cw[t][u], cx[u], acc[t]);
    }
    // (rows of x from M on are the last one again, columns from N on W's last row)
#pragma unroll
    for (int t = 0; t < NT; ++t)
        *reinterpret_cast<f32x4*>(&sums[wave][i][16 * t + 4 * q]) = acc[t];
    __syncthreads();
    if (threadIdx.x >= 32 * NT) return;
    const int m = threadIdx.x / (2 * NT), c = 8 * (threadIdx.x % (2 * NT));
    float v[1][8] = {};
#pragma unroll
    for (int r = 0; r < WAVES; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[0][e] += sums[r][m][c + e];
    finish<T, 1>(g.e, m, 1, n0 + c, v);   // stores rows under M
}

// ───────────────────────────── rows of whole chunks ─────────────────────────────

// Rows of D 16-bit values into rows of cpr chunks of 8, zeros behind: a thread
// per chunk.
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t* x, int64_t ldx, uint4* y, int64_t chunks, int cpr, int D) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= chunks) return;
    const int64_t row = i / cpr;
    const int col = 8 * (int)(i - row * cpr), valid = D - col;
    const uint16_t* p = x + row * ldx + col;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (valid >= 8) {
        __builtin_memcpy(w, p, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < valid) w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    }
    y[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// ───────────────────────────── dz and the bias gradient ─────────────────────────────

// Adds the remainders of eight values.
template <typename T>
__device__ __forceinline__ void load_rem8(const uint8_t* p, int valid, float (&v)[8]) {
    uint32_t w[2] = {0u, 0u};
    if (valid >= 8) {
        __builtin_memcpy(w, p, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = with_rem<T>(v[i], (w[i >> 2] >> (8 * (i & 3))) & 0xffu);
}

struct DactArgs {
    const void* dy;
    int64_t lddy;
    int dy32;
    const void* kept;       // [M, N]: y = relu(z)² (from_y), or what the forward's aux holds; null: codes or no activation
    const uint8_t* rem;     // [M, N]: its next 8 bits
    int from_y;
    const int8_t* codes;    // checkpoint of z
    const uint8_t* scales;
    int act;
    void* dz;               // [M, ldz] or null
    int64_t ldz;            // >= N; columns from N on are written as zeros
    float* part;            // [gridDim.y][N] column sums, or null
    int64_t M;
    int N;
};

// dz = dy·act'(z), rounded to the operands' type: both products that read it run
// on 16-bit matrix instructions, and 32 bits would cost them twice the time or
// more.  dx and dW are off by √2 of a 16-bit result's own rounding for it; db sums
// the values before.  In chunks of 8 columns: TX chunks across, 256/TX rows down
// a block, rows strided over gridDim.y, two of them loaded at a time
// (8192 x 8192 bf16 relu² from y: 4.96 TB/s; four at a time, on fewer waves, 3.97).
template <typename T>
__global__ __launch_bounds__(256) void dact_kernel(DactArgs a, int TX) {
    constexpr int U = 2;
    __shared__ float sums[256 * 8];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, TY = 256 / TX;
    const int col = 8 * (blockIdx.x * TX + tx), valid = a.N - col;
    const int64_t step = (int64_t)gridDim.y * TY, np = padded(a.N);
    float s[8] = {};
    if (col < a.ldz || valid > 0) {
        for (int64_t first = (int64_t)blockIdx.y * TY + ty; first < a.M; first += U * step) {
            float d[U][8], z[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = first + u * step;
                if (row >= a.M) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] = z[u][i] = 0.0f;
                    continue;
                }
                if (a.dy32)
                    load8(reinterpret_cast<const float*>(a.dy) + row * a.lddy + col, valid, d[u]);
                else
                    load8(reinterpret_cast<const T*>(a.dy) + row * a.lddy + col, valid, d[u]);
                if (a.act == ACT_NONE) continue;
                if (a.codes) {
                    const int64_t at = row * np + (valid > 0 ? col : 0);
                    decode8(*reinterpret_cast<const uint2*>(a.codes + at), a.scales[at / GROUP], z[u]);
                } else {
                    load8(reinterpret_cast<const T*>(a.kept) + row * a.N + col, valid, z[u]);
                    load_rem8<T>(a.rem + row * a.N + col, valid, z[u]);
                }
            }
            // the factor of dy
            if (a.act == ACT_RELU2 && a.from_y) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] *= 2.0f * __builtin_amdgcn_sqrtf(z[u][i]);
            } else if (a.act == ACT_RELU2) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] *= z[u][i] < 0.0f ? 0.0f : 2.0f * z[u][i];   // a NaN stays one
            } else if (a.act != ACT_NONE) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] *= a.act == ACT_TANH ? tanh_slope(z[u][i]) : sigmoid_slope(z[u][i]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = first + u * step;
                if (row >= a.M) continue;
                if (valid < 8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] = i < valid ? d[u][i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += d[u][i];
                if (a.dz) store8(reinterpret_cast<T*>(a.dz) + row * a.ldz + col, (int)min(a.ldz - col, (int64_t)8), d[u]);
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i * 256 + threadIdx.x] = s[i];
    __syncthreads();
    if (ty != 0) return;
    for (int r = 1; r < TY; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += sums[i * 256 + r * TX + tx];
    if (valid > 0) store8(a.part + (int64_t)blockIdx.y * a.N + col, valid, s);
}

// Column sums of part [G][N], in order within 16 interleaved runs of rows.
template <typename T>
__global__ __launch_bounds__(256) void bias_reduce_kernel(const float* part, int G, int N, T* out) {
    __shared__ float s[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + c;
    float t = 0.0f;
    if (col < N) {
#pragma unroll 8
        for (int g = r; g < G; g += 16) t += part[(int64_t)g * N + col];
    }
    s[r][c] = t;
    __syncthreads();
    if (r != 0 || col >= N) return;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += s[i][c];
    out[col] = (T)sum;
}

rwkv_status status_of(const char* what) {
    const hipError_t e = hipGetLastError();
    RWKV_REQUIRE(e == hipSuccess, RWKV_E_HIP, "%s: %s", what, hipGetErrorString(e));
    return RWKV_OK;
}

// ───────────────────────────── routes ─────────────────────────────

struct Route {
    int bm, bn;       // output tile
    int64_t full;     // tiles taken whole
    int splits, per;  // K ranges of the others
};

int64_t tiles_of(int64_t M, int64_t N, int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

// Microseconds of the output tiles, fitted to 3186 timings of 216 sizes (16 ..
// 8192 rows, 96 .. 8192 columns, K 512 .. 8192), each tile in 1 .. 32 ranges of
// K: a CU that takes n pieces of `stages` each needs
//   start·⌈n / fit⌉ + stages·(first + more·(n − 1))·(1 + 0.23·share of busy CUs).
// The cheapest of the four is 0.8 % behind the fastest one measured, in the mean.
// A K below 512, which lies outside the fit, costs more than this says: output
// bytes have no term (8192 x 2048 x 96 by 64 x 64 tiles: 7.4 us here, 21 measured).
struct Shape {
    int bm, bn, fit;
    double start, first, more;
};
constexpr Shape SHAPES[] = {{256, 256, 1, 8.5, 1.10, 1.15}, {256, 128, 1, 2.8, 0.70, 0.73},
                            {128, 128, 2, 1.8, 0.41, 0.40}, {64, 64, 4, 0.3, 0.245, 0.152}};

double pieces_cost(const Shape& s, int64_t pieces, int stages, bool odd) {
    if (pieces == 0) return 0;
    const int64_t n = (pieces + 255) / 256;
    const double busy = std::min(1.0, pieces / 256.0);
    const double wait = odd ? 0.25 : 0.0;   // misaligned loads take longer
    return s.start * ((n + s.fit - 1) / s.fit) + stages * (s.first + wait + s.more * (n - 1)) * (1 + 0.23 * busy);
}

// The tile, and how many of its tiles are taken whole: all; or whole rounds of
// the 256 CUs, with the rest in ranges of K, for whose sums a second launch
// (3.3 us) reads and writes 4 bytes a value and range at 6.4 TB/s.  km: both
// operands k-major, for which the largest tile has no kernel for ranges (it
// would spill registers, whose reloads wait for every load before them).
Route route_of(int64_t M, int64_t N, int64_t K, bool odd, bool km) {
    const int nst = (int)((K + BK - 1) / BK);
    Route best{};
    double least = 1e300;
    for (const Shape& s : SHAPES) {
        if (odd && s.bm == 256) continue;   // its loads want aligned rows
        const int64_t tiles = tiles_of(M, N, s.bm, s.bn);
        const double whole = pieces_cost(s, tiles, nst, odd);
        if (whole < least) least = whole, best = Route{s.bm, s.bn, tiles, 1, nst};
        const int64_t round = s.fit > 1 ? tiles : 256, full = odd || tiles < 256 ? 0 : tiles / round * round, rest = tiles - full;
        if (rest == 0 || rest > 256 || (km && s.bn == 256)) continue;
        const double before = full ? pieces_cost(s, full, nst, odd) + 4 : 0;
        for (int split = 2; split <= 32 && split * 2 <= nst; split = split < 4 ? split + 1 : split * 2) {
            const int per = (nst + split - 1) / split, splits = (nst + per - 1) / per;
            const double t = before + pieces_cost(s, rest * splits, per, odd) + 3.3 + (double)(rest * splits) * s.bm * s.bn * 8 / 6.4e6;
            if (t < least) least = t, best = Route{s.bm, s.bn, full, splits, per};
        }
    }
    return best;
}

int64_t route_workspace(const Route& r, int64_t M, int64_t N) {
    const int64_t rest = tiles_of(M, N, r.bm, r.bn) - r.full;
    return rest * r.splits * r.bm * r.bn * 4;
}

// The whole tiles, then the pieces of the others, on at most `fit` workgroups
// (what the LDS of 256 CUs holds).
template <typename T, bool AKM, bool BKM, int AM, int AN>
void gemm_launch_dma(int fit, const GemmArgs& g, int64_t items, hipStream_t s) {
    const dim3 whole((unsigned)std::min<int64_t>(g.full, fit)), pieces((unsigned)std::min<int64_t>(items - g.full, fit));
    if (g.full > 0) {
        if constexpr (!AKM && !BKM) {
            if (g.e.plain) rwkv::launch(gemm_dma_kernel<T, AKM, BKM, 2, 2, AM, AN, EPI_PLAIN>, whole, dim3(256), s, g);
            else rwkv::launch(gemm_dma_kernel<T, AKM, BKM, 2, 2, AM, AN, EPI_FULL>, whole, dim3(256), s, g);
        } else {
            rwkv::launch(gemm_dma_kernel<T, AKM, BKM, 2, 2, AM, AN, EPI_PLAIN>, whole, dim3(256), s, g);
        }
    }
    if constexpr (!(AKM && BKM && AN == 8))
        if (items > g.full) rwkv::launch(gemm_dma_kernel<T, AKM, BKM, 2, 2, AM, AN, EPI_PART>, pieces, dim3(256), s, g);
}

template <typename T, bool AKM, bool BKM, bool ODD>
void gemm_launch_tile(const Route& r, const GemmArgs& g, hipStream_t s) {
    const int64_t items = g.full + (tiles_of(g.M, g.N, r.bm, r.bn) - g.full) * g.splits;
    const dim3 grid((unsigned)items);
    if constexpr (!ODD) {
        if (r.bm == 256 && r.bn == 256) return gemm_launch_dma<T, AKM, BKM, 8, 8>(256, g, items, s);
        if (r.bm == 256) return gemm_launch_dma<T, AKM, BKM, 8, 4>(256, g, items, s);
        if (r.bm == 128) return gemm_launch_dma<T, AKM, BKM, 4, 4>(512, g, items, s);
    }
    if (r.bm == 128)
        rwkv::launch(gemm_kernel<T, AKM, BKM, 2, 2, 4, 4, true>, grid, dim3(256), s, g);
    else
        rwkv::launch(gemm_kernel<T, AKM, BKM, 2, 2, 2, 2, ODD>, grid, dim3(256), s, g);
}

// Few rows with a short K (a wave's loads on their way at once hold 2048 of it,
// 1024 with codes), or with two blocks of columns per CU; elsewhere x's loads
// cost as much as W's and ranges of K are faster.  us by rows16_kernel, by 64 x
// 64 tiles (bf16, back to back, W from memory):
//   N      K      1 row        16 rows          N      K      1 row       16 rows
//   1024   1024   4.4,  8.4     4.9,  8.5       4096   4096   9.0, 16.3   11.8, 16.8
//   4096   1024   4.7,  9.3     5.1,  8.6       4096   8192  18.9, 19.3   22.7, 19.7
//   8192   2048  10.6, 22.8    12.5, 22.7      14336   4096  26.5, 45.1   38.9, 45.3
//   8192    512   6.6,  5.7     7.0,  5.7      14336   8192  54.8, 51.5   76.6, 53.3
// The rule errs both ways: K = 2048 of fewer columns would gain as well (4096 x
// 2048 6.4 and 11.3), and from N = 6144 on a K of 512, or one of 8192, loses.
bool rows16_applies(int64_t M, int64_t N, int64_t K) { return M <= 16 && (K <= 1024 || N >= 8192); }

// C = A·Bᵀ by the route of its sizes, then the epilogue.
rwkv_status gemm_run(const char* what, bool akm, bool bkm, int dt, GemmArgs g, void* workspace, int64_t bytes,
                     hipStream_t s) {
    if (!akm && !bkm && rows16_applies(g.M, g.N, g.K)) {
        const int nt = g.e.codes ? 2 : 1;   // a group of codes is 32 columns
        const dim3 grid((unsigned)((g.N + 16 * nt - 1) / (16 * nt)));
        if (dt == RWKV_BF16 && nt == 1) rwkv::launch(rows16_kernel<bf16, 1>, grid, dim3(512), s, g);
        else if (dt == RWKV_BF16) rwkv::launch(rows16_kernel<bf16, 2>, grid, dim3(512), s, g);
        else if (nt == 1) rwkv::launch(rows16_kernel<f16, 1>, grid, dim3(512), s, g);
        else rwkv::launch(rows16_kernel<f16, 2>, grid, dim3(512), s, g);
        return status_of(what);
    }
    const bool aligned = (uintptr_t)g.a % 16 == 0 && (uintptr_t)g.b % 16 == 0 && g.lda % 8 == 0 && g.ldb % 8 == 0;
    const bool odd = !aligned || ((!akm || !bkm) && g.K % 8 != 0);
    const Route r = route_of(g.M, g.N, g.K, odd, akm && bkm);
    const int64_t tiles = tiles_of(g.M, g.N, r.bm, r.bn), rest = tiles - r.full;
    RWKV_REQUIRE(r.full + rest * r.splits < (int64_t(1) << 22), RWKV_E_SHAPE, "%s: too many output tiles", what);
    const int64_t need = route_workspace(r, g.M, g.N);
    RWKV_REQUIRE(need == 0 || (workspace && bytes >= need && (uintptr_t)workspace % 16 == 0), RWKV_E_SHAPE,
                 "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)need);
    g.full = (int)r.full;
    g.splits = r.splits;
    g.per = r.per;
    g.part = (float*)workspace;
    g.e.plain = !g.e.bias && !g.e.res && !g.e.wide && !g.e.aux && !g.e.rem && !g.e.codes && g.e.act == ACT_NONE;
    auto by_layout = [&](auto type, auto o) {
        using T = decltype(type);
        constexpr bool O = decltype(o)::value;
        if (!akm && !bkm) gemm_launch_tile<T, false, false, O>(r, g, s);
        else if (!akm) gemm_launch_tile<T, false, true, O>(r, g, s);
        else gemm_launch_tile<T, true, true, O>(r, g, s);
        if (rest > 0)
            rwkv::launch(split_reduce_kernel<T>, dim3((unsigned)(rest * (r.bm * r.bn / 2048))), dim3(256), s, g, r.bm, r.bn,
                         (int)((g.M + r.bm - 1) / r.bm), (int)((g.N + r.bn - 1) / r.bn));
    };
    if (dt == RWKV_BF16 && odd) by_layout(bf16{}, std::true_type{});
    else if (dt == RWKV_BF16) by_layout(bf16{}, std::false_type{});
    else if (odd) by_layout(f16{}, std::true_type{});
    else by_layout(f16{}, std::false_type{});
    return status_of(what);
}

// For either kind of alignment (the pointers are not known yet).
int64_t gemm_workspace(int64_t M, int64_t N, int64_t K, bool km) {
    if (M == 0) return 0;
    return std::max(route_workspace(route_of(M, N, K, false, km), M, N), route_workspace(route_of(M, N, K, true, km), M, N));
}

bool shape_ok(int64_t M, int64_t N, int64_t K) {
    return M >= 0 && M <= (1 << 24) && N >= 1 && N <= (1 << 20) && K >= 1 && K <= (1 << 20);
}
bool half_ok(int dt) { return dt == RWKV_BF16 || dt == RWKV_F16; }
bool ld_ok(int64_t ld, int64_t cols) { return ld >= cols && ld <= MAX_LD; }

// Blocks of dact_kernel: 2048 at most, half of that with db, to which each
// block down the rows adds one partial row.
void dact_geometry(int64_t M, int64_t N, bool db, int& TX, int& gx, int& gy) {
    const int64_t chunks = (N + 7) / 8;
    TX = 1;
    while (TX < 64 && TX < chunks) TX *= 2;
    gx = (int)((chunks + TX - 1) / TX);
    const int ty = 256 / TX;
    gy = (int)std::max<int64_t>(1, std::min<int64_t>((M + ty - 1) / ty, std::max(1, (db ? 1024 : 2048) / gx)));
}

}  // namespace

extern "C" {

int64_t rwkv_linear_fwd_workspace(int64_t M, int64_t N, int64_t K) {
    return shape_ok(M, N, K) && !rows16_applies(M, N, K) ? gemm_workspace(M, N, K, false) : 0;
}

rwkv_status rwkv_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                            const void* residual, int64_t ldr, void* y, rwkv_dtype y_dt, void* aux, uint8_t* rem,
                            int8_t* codes, uint8_t* scales, rwkv_activation act, rwkv_dtype dt, int64_t M, int64_t N, int64_t K,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    RWKV_REQUIRE(half_ok(dt) && (y_dt == dt || y_dt == RWKV_F32), RWKV_E_DTYPE, "linear_fwd: types %d, output %d",
                 (int)dt, (int)y_dt);
    RWKV_REQUIRE(act >= 0 && act <= ACT_SIGMOID, RWKV_E_UNSUPPORTED, "linear_fwd: activation %d", (int)act);
    RWKV_REQUIRE(shape_ok(M, N, K) && ld_ok(ldx, K) && ld_ok(ldw, K) && (!residual || ldr >= N), RWKV_E_SHAPE,
                 "linear_fwd: M=%lld N=%lld K=%lld ldx=%lld ldw=%lld ldr=%lld", (long long)M, (long long)N,
                 (long long)K, (long long)ldx, (long long)ldw, (long long)ldr);
    RWKV_REQUIRE(M == 0 || (x && w && y), RWKV_E_NULL, "linear_fwd: null buffer");
    RWKV_REQUIRE(!codes == !scales, RWKV_E_NULL, "linear_fwd: codes and scales go together");
    RWKV_REQUIRE(!aux || rem, RWKV_E_NULL, "linear_fwd: aux without its remainders");
    RWKV_REQUIRE(!rem || aux || (act == ACT_RELU2 && y_dt == dt && !residual), RWKV_E_UNSUPPORTED,
                 "linear_fwd: remainders of a y that is not relu(z)^2, of another type, or with a residual in it");
    if (M == 0) return RWKV_OK;
    GemmArgs g{};
    g.a = x, g.lda = ldx, g.b = w, g.ldb = ldw, g.M = M, g.N = (int)N, g.K = g.KB = (int)K;
    g.e = Epilogue{bias, residual, ldr, y, y_dt == RWKV_F32, aux, rem, codes, scales, (int)act, M, (int)N};
    return gemm_run("linear_fwd", false, false, dt, g, workspace, workspace_bytes, (hipStream_t)stream);
}

rwkv_status rwkv_linear_pad(const void* x, int64_t ldx, void* y, int64_t N, int64_t D, void* stream) {
    RWKV_REQUIRE(N >= 0 && N <= (1 << 24) && D >= 1 && D <= (1 << 20) && ldx >= D, RWKV_E_SHAPE,
                 "linear_pad: N=%lld D=%lld ldx=%lld", (long long)N, (long long)D, (long long)ldx);
    RWKV_REQUIRE(N == 0 || (x && y && (uintptr_t)y % 16 == 0), RWKV_E_NULL, "linear_pad: null or misaligned buffer");
    if (N == 0) return RWKV_OK;
    const int64_t cpr = (D + 7) / 8, chunks = N * cpr, blocks = (chunks + 255) / 256;
    RWKV_REQUIRE(blocks < (int64_t(1) << 31), RWKV_E_SHAPE, "linear_pad: %lld values", (long long)(N * D));
    rwkv::launch(pad_kernel, dim3((unsigned)blocks), dim3(256), (hipStream_t)stream, (const uint16_t*)x, ldx, (uint4*)y, chunks,
                 (int)cpr, (int)D);
    return status_of("linear_pad launch");
}

int64_t rwkv_linear_dact_workspace(int64_t M, int64_t N) {
    if (!shape_ok(M, N, 1)) return 0;
    int TX, gx, gy;
    dact_geometry(M, N, true, TX, gx, gy);
    return (int64_t)gy * N * 4;
}

rwkv_status rwkv_linear_dact(const void* dy, int64_t lddy, rwkv_dtype dy_dt, const void* kept,
                             const uint8_t* rem, int kept_is_y, const int8_t* codes, const uint8_t* scales,
                             rwkv_activation act, void* dz, int64_t ldz, void* db, rwkv_dtype dt, int64_t M, int64_t N, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    RWKV_REQUIRE(half_ok(dt) && (dy_dt == dt || dy_dt == RWKV_F32), RWKV_E_DTYPE, "linear_dact: types %d, dy %d",
                 (int)dt, (int)dy_dt);
    RWKV_REQUIRE(act >= 0 && act <= ACT_SIGMOID && (!kept_is_y || act == ACT_RELU2), RWKV_E_UNSUPPORTED,
                 "linear_dact: activation %d, kept_is_y %d", (int)act, kept_is_y);
    RWKV_REQUIRE(shape_ok(M, N, 1) && lddy >= N && (!dz || (ldz >= N && ldz < N + 8)), RWKV_E_SHAPE,
                 "linear_dact: M=%lld N=%lld lddy=%lld ldz=%lld", (long long)M, (long long)N, (long long)lddy,
                 (long long)ldz);
    RWKV_REQUIRE(!codes == !scales && !(codes && kept), RWKV_E_NULL,
                 "linear_dact: codes and scales go together, without kept");
    RWKV_REQUIRE(!kept == !rem, RWKV_E_NULL, "linear_dact: kept and its remainders go together");
    RWKV_REQUIRE(M == 0 || (dy && (act == ACT_NONE || kept || codes)), RWKV_E_NULL, "linear_dact: null buffer");
    int TX, gx, gy;
    dact_geometry(M, N, db != nullptr, TX, gx, gy);
    RWKV_REQUIRE(!db || (workspace && workspace_bytes >= (int64_t)gy * N * 4 && (uintptr_t)workspace % 16 == 0),
                 RWKV_E_SHAPE, "linear_dact: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                 (long long)gy * N * 4);
    if (!db && !dz) return RWKV_OK;
    const hipStream_t s = (hipStream_t)stream;
    const DactArgs a{dy, lddy, dy_dt == RWKV_F32, kept, rem, kept_is_y, codes, scales, (int)act, dz, dz ? ldz : N,
                     db ? (float*)workspace : nullptr, M, (int)N};
    // a pitch may reach into the chunk after N's last: its zeros are written too
    const unsigned across = (unsigned)((a.ldz + 8 * TX - 1) / (8 * TX));
    const dim3 grid(across, (unsigned)gy), bgrid((unsigned)((N + 15) / 16));
    if (dt == RWKV_BF16) {
        rwkv::launch(dact_kernel<bf16>, grid, dim3(256), s, a, TX);
        if (db) rwkv::launch(bias_reduce_kernel<bf16>, bgrid, dim3(256), s, (const float*)workspace, gy, (int)N, (bf16*)db);
    } else {
        rwkv::launch(dact_kernel<f16>, grid, dim3(256), s, a, TX);
        if (db) rwkv::launch(bias_reduce_kernel<f16>, bgrid, dim3(256), s, (const float*)workspace, gy, (int)N, (f16*)db);
    }
    return status_of("linear_dact launch");
}

int64_t rwkv_linear_dgrad_workspace(int64_t M, int64_t N, int64_t K) {
    return shape_ok(M, N, K) ? gemm_workspace(M, K, N, false) : 0;
}

rwkv_status rwkv_linear_dgrad(const void* dz, int64_t ldz, const void* w, int64_t ldw, void* dx, rwkv_dtype dt,
                              int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    RWKV_REQUIRE(half_ok(dt), RWKV_E_DTYPE, "linear_dgrad: dtype %d", (int)dt);
    RWKV_REQUIRE(shape_ok(M, N, K) && ld_ok(ldz, N) && ld_ok(ldw, K), RWKV_E_SHAPE,
                 "linear_dgrad: M=%lld N=%lld K=%lld ldz=%lld ldw=%lld", (long long)M, (long long)N, (long long)K,
                 (long long)ldz, (long long)ldw);
    RWKV_REQUIRE(M == 0 || (dz && w && dx), RWKV_E_NULL, "linear_dgrad: null buffer");
    if (M == 0) return RWKV_OK;
    GemmArgs g{};
    // the pitch's columns beyond N hold zeros (rwkv_linear_dact writes them),
    // and W has no rows there: contract over the multiple of 8
    const int64_t kk = ldz >= (N + 7) / 8 * 8 ? (N + 7) / 8 * 8 : N;
    g.a = dz, g.lda = ldz, g.b = w, g.ldb = ldw, g.M = M, g.N = (int)K, g.K = (int)kk, g.KB = (int)N;
    g.e = Epilogue{nullptr, nullptr, 0, dx, 0, nullptr, nullptr, nullptr, nullptr, ACT_NONE, M, (int)K};
    return gemm_run("linear_dgrad", false, true, dt, g, workspace, workspace_bytes, (hipStream_t)stream);
}

int64_t rwkv_linear_wgrad_workspace(int64_t M, int64_t N, int64_t K) {
    return shape_ok(M, N, K) && M > 0 ? gemm_workspace(N, K, M, true) : 0;
}

rwkv_status rwkv_linear_wgrad(const void* dz, int64_t ldz, const void* x, int64_t ldx, void* dw, rwkv_dtype dt,
                              int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    RWKV_REQUIRE(half_ok(dt), RWKV_E_DTYPE, "linear_wgrad: dtype %d", (int)dt);
    RWKV_REQUIRE(shape_ok(M, N, K) && M >= 1 && ld_ok(ldz, N) && ld_ok(ldx, K), RWKV_E_SHAPE,
                 "linear_wgrad: M=%lld N=%lld K=%lld ldz=%lld ldx=%lld", (long long)M, (long long)N, (long long)K,
                 (long long)ldz, (long long)ldx);
    RWKV_REQUIRE(dz && x && dw, RWKV_E_NULL, "linear_wgrad: null buffer");
    GemmArgs g{};
    g.a = dz, g.lda = ldz, g.b = x, g.ldb = ldx, g.M = N, g.N = (int)K, g.K = g.KB = (int)M;
    g.e = Epilogue{nullptr, nullptr, 0, dw, 0, nullptr, nullptr, nullptr, nullptr, ACT_NONE, N, (int)K};
    return gemm_run("linear_wgrad", true, true, dt, g, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
