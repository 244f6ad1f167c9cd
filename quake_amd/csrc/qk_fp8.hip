// 8-bit state stores and the products over them (gfx950): e4m3 codes with one power-of-two scale for each block of 128
// amplitudes.
//
//   write     psi -> codes, scales, gains            code = e4m3(component * 2^-e), e = the least integer with
//                                                    max |component of the block| * 2^-e <= 448
//   read      codes, scales -> code * 2^e
//   gram8     K_ij = gain_i gain_j |sum_b conj(q_i[b]) q_j[b]|^2,  gain = ||psi||^2 / ||q||^2
//   decision8 out[m][c] = sum_j K_mj coef[j][c] + intercept[c], K not written (but for a few long rows)
//
// A row of D amplitudes is laid out as chunks of 64 amplitudes: 64 real codes, then 64 imaginary codes (128 bytes, one
// cache line); the last chunk is padded with zero codes.  Two chunks share one scale byte e + 127.  Scales are powers of
// two because that is exact: multiplying by one never rounds, and an e4m3 code has the same relative step whatever the
// scale (the scale only keeps the block inside the format's 2^18 range).
//
// Arithmetic of the products, one form for every type of K and every kernel: codes are widened to bf16 (exact: e4m3 has 4
// significant bits, bf16 has 8 and FP32's exponents) with the block's scale applied in the same instruction; a product of two codes
// is exact in FP32, sums are FP32, K is converted to its type once.  The 8-bit matrix instruction is not used: it aligns groups of 8
// products to the largest and cuts what falls below about 13 bits of it, which leaves K of similar states 1e-4 low and small entries
// (sums that cancel) off by a per cent.  Rates measured from registers: 8-bit instruction 4.2 .. 4.8 PFLOP/s, bf16 2.49, bf16
// with two widening instructions each 1.82.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <new>
#include <vector>

#include "qk_common.h"

namespace qk {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;            // amplitudes per chunk
constexpr int kChunkBytes = 128;
constexpr int kBlock = 128;           // amplitudes per scale
constexpr int64_t kThreads = 0xffffffffLL;      // of a launch: one with more does not fail, it wraps around
constexpr int kGram8Jobs = 24;        // jobs of one launch (their records travel as kernel arguments: under 4 KiB)

static inline int64_t code_bytes(int64_t D) { return (D + kChunk - 1) / kChunk * kChunkBytes; }
static inline int64_t scale_bytes(int64_t D) { return ((D + kBlock - 1) / kBlock + 3) / 4 * 4; }

// ---- write -------------------------------------------------------------------------------------------------------------
// FP64 -> FP32 rounding to odd: a value that FP32 does not hold exactly gets its last bit set after truncation, so a
// second rounding to e4m3 gives what rounding the FP64 value once would have given.
__device__ __forceinline__ float to_f32_odd(double v) {
    float f = (float)v;
    const double r = (double)f;
    uint32_t u = __float_as_uint(f);
    if (fabs(r) > fabs(v)) u -= 1;
    if (r != v) u |= 1;
    return (v != v || fabs(r) == __builtin_huge_val()) ? __builtin_nanf("") : __uint_as_float(u);
}
__device__ __forceinline__ float to_f32_odd(float v) { return fabsf(v) < __builtin_huge_valf() ? v : __builtin_nanf(""); }

// e of a block whose largest component is `top` >= 0 (448 = 1.75 * 2^8); no less than -100, so that code * 2^e is a normal
// number in FP32 and bf16
__device__ __forceinline__ int scale_exponent(float top) {
    const uint32_t u = __float_as_uint(top);
    if (u == 0) return 0;
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(-100, e);
}

template <typename T> struct Pair;
template <> struct Pair<double> { typedef double2 type; };
template <> struct Pair<float> { typedef float2 type; };

// Largest of 32 lanes, in all of them
__device__ __forceinline__ float half_max(float v) {
#define QK_MAX_DPP(CTRL) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)))
    QK_MAX_DPP(0xB1);      // neighbours in pairs,
    QK_MAX_DPP(0x4E);      // pairs in fours,
    QK_MAX_DPP(0x141);     // fours in eights (mirrored),
    QK_MAX_DPP(0x140);     // eights in sixteens (mirrored)
#undef QK_MAX_DPP
    return fmaxf(v, __shfl_xor(v, 16, 64));
}

// Four lanes of a quad, byte k of lane l -> byte l of lane k
__device__ __forceinline__ uint32_t quad_transpose(uint32_t v, int lane) {
    const uint32_t x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);
    v = __builtin_amdgcn_perm(x, v, lane & 1 ? 0x03070105u : 0x06020400u);      // bytes 0 .. 3: own, 4 .. 7: the neighbour's
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);
    return __builtin_amdgcn_perm(y, v, lane & 2 ? 0x03020706u : 0x05040100u);
}

// One half-wave (32 lanes) holds one block: lane i has amplitudes i, i + 32, i + 64, i + 96 (coalesced loads, the next
// block's in flight while one is rounded) and, after a transpose in its quad, stores the codes of four neighbours at once.  WPR
// waves work on one row and its sums meet in LDS.  Memory bound: 4096 rows of 65536 complex128 amplitudes 953 us, 5.05 TB/s read and
// written (a large copy reaches 4.84, a read 6.1).
template <typename T, int WPR>
__global__ __launch_bounds__(WPR < 4 ? 256 : 64 * WPR) void states8_write_kernel(const void* psi_, int64_t N, int64_t D, int64_t ld,
                                                                                uint8_t* codes, uint8_t* scales, float* gains) {
    constexpr int WAVES = WPR < 4 ? 4 : WPR;
    constexpr int ROWS = WAVES / WPR;
    __shared__ double part[2][WAVES];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, i = lane & 31;
    const int64_t row = (int64_t)blockIdx.x * ROWS + wave / WPR;
    const int sub = wave % WPR;
    const int64_t cb = (D + kChunk - 1) / kChunk * kChunkBytes, blocks = (D + kBlock - 1) / kBlock, sb = (blocks + 3) / 4 * 4;
    typedef typename Pair<T>::type P;
    double norm = 0.0, kept = 0.0;
    if (row < N) {
        const P* src = (const P*)psi_ + row * ld;
        uint8_t* dst = codes + row * cb;
        uint8_t* sc = scales + row * sb;
        P v[4];
        auto load = [&](int64_t b) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t at = b * kBlock + 32 * k + i;
                v[k].x = v[k].y = 0;
                if (at < D) v[k] = src[at];
            }
        };
        load(2 * sub + half);
        for (int64_t b0 = 2 * sub; b0 < sb; b0 += 2 * WPR) {
            const int64_t b = b0 + half;
            float re[4], im[4], top = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                norm += (double)v[k].x * (double)v[k].x + (double)v[k].y * (double)v[k].y;
                re[k] = to_f32_odd(v[k].x);
                im[k] = to_f32_odd(v[k].y);
                top = fmaxf(top, fmaxf(fabsf(re[k]), fabsf(im[k])));      // (fmax drops NaN)
            }
            if (b0 + 2 * WPR < sb) load(b + 2 * WPR);
            const int e = scale_exponent(half_max(top));
            uint32_t wr = 0, wi = 0;      // byte k: the code of amplitude 32 k + i
            double sq = 0.0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = ldexpf(re[k], -e), c = ldexpf(im[k], -e);
                uint32_t p = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, c, 0, false) & 0xffffu;
                p &= ~(((p & 0x7f7fu) + 0x0101u) & 0x8080u);      // one code for NaN: 0x7f
                wr |= (p & 0xffu) << (8 * k);
                wi |= ((p >> 8) & 0xffu) << (8 * k);
                const double qa = __builtin_amdgcn_cvt_f32_fp8((int)p, 0), qc = __builtin_amdgcn_cvt_f32_fp8((int)p, 1);
                sq += qa * qa + qc * qc;
            }
            kept += ldexp(sq, 2 * e);
            wr = quad_transpose(wr, lane);
            wi = quad_transpose(wi, lane);
            const int64_t at = b * kBlock + 32 * (i & 3) + (i & ~3);      // four amplitudes from here on
            const int64_t o = (at >> 6) * kChunkBytes + (at & 63);
            if (o < cb) {
                *(uint32_t*)(dst + o) = wr;
                *(uint32_t*)(dst + o + kChunk) = wi;
            }
            if (i == 0) sc[b] = (uint8_t)(b < blocks ? e + 127 : 127);
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
            norm += __shfl_xor(norm, m, 64);
            kept += __shfl_xor(kept, m, 64);
        }
    }
    if (lane == 0) {
        part[0][wave] = norm;
        part[1][wave] = kept;
    }
    __syncthreads();
    if (row < N && sub == 0 && lane == 0) {
        double n = 0.0, q = 0.0;
        for (int w = 0; w < WPR; ++w) {
            n += part[0][wave + w];
            q += part[1][wave + w];
        }
        gains[row] = q == 0.0 ? 0.f : (float)(n / q);
    }
}

// ---- read --------------------------------------------------------------------------------------------------------------
// Rows of 512 amplitudes or more: a wave takes 512 of them, whose codes are 1024 bytes in a row and whose scales are one
// dword: one load of 16 bytes per lane, through LDS to pairs of amplitudes, four stores of whole lines.  A row number outside
// 0 .. of - 1 gives a row of NaN.  VEC: rows of psi start on 16 bytes.  Memory bound, mostly its writes: 20001 rows of 4096
// amplitudes by row number to complex64 156 us, 5.2 TB/s (2 bytes read and stored per lane, without LDS: 231 us).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void states8_read_long_kernel(const uint8_t* codes, const uint8_t* scales, const int64_t* index,
                                                                int64_t of, uint32_t items, int64_t D, void* out_, int64_t ldo,
                                                                uint32_t segments) {
    typedef typename Pair<T>::type P;
    __shared__ uint4 room[4][64];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * 4 + wave;
    if (item >= items) return;
    const int64_t cb = (D + kChunk - 1) / kChunk * kChunkBytes, sb = ((D + kBlock - 1) / kBlock + 3) / 4 * 4;
    const uint32_t n = item / segments, seg = item - n * segments;
    const int64_t row = index ? index[n] : (int64_t)n;
    const bool there = row >= 0 && row < of;
    uint4 u = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
    uint32_t e4 = 0x7f7f7f7fu;
    if (there) {
        const int64_t o = (int64_t)seg * 1024 + lane * 16;
        if (o < cb) u = *(const uint4*)(codes + row * cb + o);
        e4 = *(const uint32_t*)(scales + row * sb + seg * 4);
    }
    room[wave][lane] = u;
    __builtin_amdgcn_wave_barrier();      // (a wave's LDS accesses stay in order)
    const uint8_t* const from = (const uint8_t*)room[wave];
    P* const out = (P*)out_ + (int64_t)n * ldo + (int64_t)seg * 512;
    if constexpr (sizeof(T) == 8) {      // 16 bytes are one amplitude
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int at = k * 64 + lane, e = (int)((e4 >> (8 * (k >> 1))) & 255u) - 127;
            const int r = from[k * kChunkBytes + lane], s = from[k * kChunkBytes + kChunk + lane];
            P v;
            v.x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r, 0), e);
            v.y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s, 0), e);
            if (at < D - (int64_t)seg * 512) out[at] = v;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = k * 128 + lane * 2, b = (at >> 6) * kChunkBytes + (at & 63), e = (int)((e4 >> (8 * k)) & 255u) - 127;
        const int r = *(const uint16_t*)(from + b), s = *(const uint16_t*)(from + b + kChunk);
        P v[2];
        v[0].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r, 0), e);
        v[1].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r, 1), e);
        v[0].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s, 0), e);
        v[1].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s, 1), e);
        const int64_t left = D - (int64_t)seg * 512 - at;
        if (VEC && sizeof(T) == 4 && left > 1) *(float4*)(out + at) = make_float4((float)v[0].x, (float)v[0].y, (float)v[1].x, (float)v[1].y);
        else {
            if (left > 0) out[at] = v[0];
            if (left > 1) out[at + 1] = v[1];
        }
    }
}

// Shorter rows: a workgroup reads 2048 amplitudes (pairs of them, four pairs per thread, their loads all in flight) of as many whole rows as
// that holds.
constexpr int kReadPairs = 1024;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void states8_read_kernel(const uint8_t* codes, const uint8_t* scales, const int64_t* index,
                                                           int64_t of, int64_t N, int64_t D, void* out_, int64_t ldo, uint32_t rows) {
    typedef typename Pair<T>::type P;
    const int64_t cb = (D + kChunk - 1) / kChunk * kChunkBytes, sb = ((D + kBlock - 1) / kBlock + 3) / 4 * 4;
    const uint32_t per = (uint32_t)((D + 1) / 2);
    int64_t n[4], at[4], row[4];
    int r[4], s[4], e[4];
    bool live[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t p = k * 256 + threadIdx.x, in = p / per;
        n[k] = (int64_t)blockIdx.x * rows + in;
        at[k] = 2 * (int64_t)(p - in * per);
        live[k] = in < rows && n[k] < N;
        row[k] = live[k] ? (index ? index[n[k]] : n[k]) : -1;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool there = row[k] >= 0 && row[k] < of;
        const uint8_t* c = codes + (there ? row[k] * cb + (at[k] >> 6) * kChunkBytes + (at[k] & 63) : 0);
        e[k] = there ? (int)scales[row[k] * sb + (at[k] >> 7)] - 127 : 0;
        r[k] = there ? *(const uint16_t*)c : 0x7f7f;
        s[k] = there ? *(const uint16_t*)(c + kChunk) : 0x7f7f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!live[k]) continue;
        P* out = (P*)out_ + n[k] * ldo + at[k];
        P v[2];
        v[0].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r[k], 0), e[k]);
        v[1].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r[k], 1), e[k]);
        v[0].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s[k], 0), e[k]);
        v[1].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s[k], 1), e[k]);
        if (VEC && sizeof(T) == 4 && at[k] + 1 < D) *(float4*)out = make_float4((float)v[0].x, (float)v[0].y, (float)v[1].x, (float)v[1].y);
        else {
            out[0] = v[0];
            if (at[k] + 1 < D) out[1] = v[1];
        }
    }
}

// ---- products ----------------------------------------------------------------------------------------------------------
struct Rows8 {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* gains;
    int64_t n;
};

struct Gram8JobDev {
    Rows8 A, B;
    void* K;
    void* KT;
    int64_t ldk, ldkt;
    int64_t ws;                // first float of the job's partial sums in the workspace
    int32_t flags;
    int32_t chunks;            // chunks per row
    int32_t sb;                // scale bytes per row
    int32_t tiles_m, tiles_n;  // tile rows and columns
    int32_t slices;            // the tiles behind the first `whole` are cut into this many slices of `per` chunks,
    int32_t small;             // or (1) into 16 tiles of 32 x 32
    int32_t per;
    uint32_t live;             // tiles that have to be computed
    uint32_t whole;
    uint32_t begin;            // items of the jobs before; a job's: its whole tiles, then slice by slice the others
};

struct Gram8Args {
    Gram8JobDev job[kGram8Jobs];
    int32_t n_jobs;
    uint32_t total;            // items
    uint32_t first;            // item of the launch's first workgroup (32 x 32 tiles)
    uint32_t small;            // the items from here on are 32 x 32 tiles of the last job (launches of 128 x 128 tiles)
    float* ws;
};
static_assert(sizeof(Gram8Args) <= 4096, "kernel arguments");

// Four codes -> four bf16 values times 2^(scale - 127)
__device__ __forceinline__ void widen4(uint32_t c, float scale, v2b& lo, v2b& hi) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, scale, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, scale, true);
}
__device__ __forceinline__ v8b widen8(uint32_t c0, uint32_t c1, float scale) {
    union { v2b p[4]; v8b v; } u;
    widen4(c0, scale, u.p[0], u.p[1]);
    widen4(c1, scale, u.p[2], u.p[3]);
    return u.v;
}
__device__ __forceinline__ v8b negated(v8b v) {
    union { v8b v; uint32_t d[4]; } u;
    u.v = v;
#pragma unroll
    for (int k = 0; k < 4; ++k) u.d[k] ^= 0x80008000u;
    return u.v;
}
// 2^(byte - 127) as FP32 (a store's bytes are 27 or more)
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }

// Row of a lane's accumulator register i in a 32 x 32 tile; the column is lane & 31.
__device__ __forceinline__ int acc_row(int lane, int i) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

__device__ __forceinline__ void store_k(void* K, int64_t at, float k, int flags) {
    if (flags & QK_GRAM8_F16) ((_Float16*)K)[at] = (_Float16)k;
    else if (flags & QK_GRAM8_F64) ((double*)K)[at] = (double)k;
    else ((float*)K)[at] = k;
}

// K of an overlap and the two gains' product, in FP32 whatever K's type: which square is fused is written out, and the product is
// rounded here (the compiler would fuse it with a float16 K's conversion, in some kernels and not in others).
__device__ __forceinline__ float k_value(float re, float im, float gains) {
    float k = __builtin_fmaf(re, re, im * im) * gains;
    asm("" : "+v"(k));
    return k;
}

// One entry of K and its mirror (symmetric: the entries below the diagonal are the ones above it, so K is symmetric to the
// bit; summed on their own they would differ in the order of the imaginary part's two halves).
__device__ __forceinline__ void emit(const Gram8JobDev& J, int64_t row, int64_t col, float re, float im) {
    const bool sym = J.flags & QK_GRAM_SYMMETRIC;
    if (row >= J.A.n || col >= J.B.n || (sym && row > col)) return;
    float k = k_value(re, im, J.A.gains[row] * J.B.gains[col]);
    if (sym && row == col) k = 1.f;
    store_k(J.K, row * J.ldk + col, k, J.flags);
    if (sym && row != col) store_k(J.K, col * J.ldk + row, k, J.flags);
    if (J.KT) store_k(J.KT, col * J.ldkt + row, k, J.flags);
}

// Tile t of a job: the tiles that have to be computed, strip by strip (8 tile rows), column by column inside a strip, so
// that neighbours in the list share rows of both operands in an XCD's L2.  Symmetric: those on or above the diagonal; a
// full strip then starts with a triangle of 36.
__device__ __forceinline__ void gram8_tile(const Gram8JobDev& J, uint32_t t, uint32_t& ti, uint32_t& tj) {
    const uint32_t TM = (uint32_t)J.tiles_m, TN = (uint32_t)J.tiles_n;
    if (!(J.flags & QK_GRAM_SYMMETRIC)) {
        const uint32_t strip = t / (8u * TN), in = t - strip * 8u * TN, rows = min(8u, TM - 8u * strip);
        tj = in / rows;
        ti = 8u * strip + (in - tj * rows);
        return;
    }
    uint32_t lo = 0, hi = (TM + 7u) / 8u - 1u;             // the last strip that starts at or before t
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1u) / 2u;
        if (mid * (36u + 8u * (TM - 4u * mid - 4u)) <= t) lo = mid; else hi = mid - 1u;
    }
    uint32_t in = t - lo * (36u + 8u * (TM - 4u * lo - 4u));
    const uint32_t r0 = 8u * lo, rows = min(8u, TM - r0), tri = rows * (rows + 1u) / 2u;
    if (in < tri) {
        uint32_t c = 0;
        while (in > c) in -= ++c;                          // column c of the triangle has c + 1 tiles
        tj = r0 + c;
        ti = r0 + in;
        return;
    }
    in -= tri;
    tj = r0 + rows + in / rows;
    ti = r0 + in % rows;
}

// Item `in` of a job -> tile t, slice (-1: the whole tile)
__device__ __forceinline__ void gram8_part(const Gram8JobDev& J, uint32_t in, uint32_t& t, int& slice) {
    t = in;
    slice = -1;
    if (in >= J.whole) {
        const uint32_t cut = J.live - J.whole, k = in - J.whole;
        slice = (int)(k / cut);
        t = J.whole + (k - (uint32_t)slice * cut);
    }
}

__device__ __forceinline__ int gram8_job(const Gram8Args& a, uint32_t item) {
    int j = 0;
    while (j + 1 < a.n_jobs && a.job[j + 1].begin <= item) ++j;
    return j;
}

// re += conj(a) c, im of the same, over chunks c0, c0 + step, ... < c1 of two 32-row operands (pa, pb: this lane's rows,
// offset by its half), the next chunk's loads in flight while one is multiplied.  The matrix instruction sums 8 codes of
// either half of the wave; which 8 is free as long as both operands agree, so a lane takes whole 16-byte pieces.
struct WaveChunk {
    v4u ar[2], ai[2], br[2], bi[2];
    uint32_t ea, eb;
};
__device__ __forceinline__ void wave_load(WaveChunk& f, const uint8_t* pa, const uint8_t* sa, const uint8_t* pb, const uint8_t* sb, int c) {
    const uint8_t *a = pa + (int64_t)c * kChunkBytes, *b = pb + (int64_t)c * kChunkBytes;
    f.ea = sa[c >> 1];
    f.eb = sb[c >> 1];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        f.ar[s] = *(const v4u*)(a + 32 * s);
        f.ai[s] = *(const v4u*)(a + 64 + 32 * s);
        f.br[s] = *(const v4u*)(b + 32 * s);
        f.bi[s] = *(const v4u*)(b + 64 + 32 * s);
    }
}
__device__ __forceinline__ void wave_multiply(const WaveChunk& f, v16f& re, v16f& im) {
    const float ea = scale_value(f.ea), eb = scale_value(f.eb);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            const v8b xr = widen8(f.ar[s][q], f.ar[s][q + 1], ea), xi = widen8(f.ai[s][q], f.ai[s][q + 1], ea);
            const v8b yr = widen8(f.br[s][q], f.br[s][q + 1], eb), yi = widen8(f.bi[s][q], f.bi[s][q + 1], eb);
            re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yr, re, 0, 0, 0);
            im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yi, im, 0, 0, 0);
            re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xi, yi, re, 0, 0, 0);
            im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(negated(xi), yr, im, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);      // (widening all codes first would take twice the registers)
        }
}
__device__ __forceinline__ void wave_product(const uint8_t* pa, const uint8_t* sa, const uint8_t* pb, const uint8_t* sb, int c0,
                                             int c1, int step, v16f& re, v16f& im) {
    if (c0 >= c1) return;
    WaveChunk f, g;
    wave_load(f, pa, sa, pb, sb, c0);
    for (int c = c0;;) {
        if ((c += step) < c1) wave_load(g, pa, sa, pb, sb, c);
        wave_multiply(f, re, im);
        if (c >= c1) return;
        if ((c += step) < c1) wave_load(f, pa, sa, pb, sb, c);
        wave_multiply(g, re, im);
        if (c >= c1) return;
    }
}

// A 32 x 32 tile of a job by four waves: chunks c0 .. c1 - 1 dealt to them, their sums joined in LDS; the entries, or (ws) a
// slice's sums.
__device__ __forceinline__ void wave_tile(const Gram8JobDev& J, int64_t row, int64_t col, int c0, int c1, float (*part)[32][64], float2* ws) {
    constexpr int W = 4;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int64_t cb = (int64_t)J.chunks * kChunkBytes;
    const int64_t ra = min(row + r, J.A.n - 1), rb = min(col + r, J.B.n - 1);
    v16f re, im;
#pragma unroll
    for (int i = 0; i < 16; ++i) re[i] = im[i] = 0.f;
    wave_product(J.A.codes + ra * cb + 16 * h, J.A.scales + ra * J.sb, J.B.codes + rb * cb + 16 * h, J.B.scales + rb * J.sb, c0 + wave,
                 c1, W, re, im);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        part[wave][i][lane] = re[i];
        part[wave][16 + i][lane] = im[i];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16 / W; ++k) {
        const int i = wave * (16 / W) + k;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            x += part[w][i][lane];
            y += part[w][16 + i][lane];
        }
        if (ws) ws[i * 64 + lane] = make_float2(x, y);
        else emit(J, row + acc_row(lane, i), col + r, x, y);
    }
}

// One tile or slice per workgroup.  Latency bound, a launch and the trip of its first loads: 100 rows of 16 amplitudes 4.7 us on the GPU, 10
// from call to call; 24 kernels of 100 rows and 16 to 1024 amplitudes 9 to 15 us.
__global__ __launch_bounds__(256, 3) void gram8_wave_kernel(Gram8Args args) {
    __shared__ float part[4][32][64];
    const uint32_t item = args.first + blockIdx.x;
    const Gram8JobDev& J = args.job[gram8_job(args, item)];
    uint32_t t, ti, tj;
    int slice;
    gram8_part(J, item - J.begin, t, slice);
    gram8_tile(J, t, ti, tj);
    const int c0 = max(slice, 0) * J.per, c1 = slice < 0 ? J.chunks : min(J.chunks, c0 + J.per);
    wave_tile(J, (int64_t)ti * 32, (int64_t)tj * 32, c0, c1, part,
              slice < 0 ? nullptr : (float2*)(args.ws + J.ws) + ((int64_t)(t - J.whole) * J.slices + slice) * 1024);
}

// ---- few rows against many ---------------------------------------------------------------------------------------------
// Up to 32 rows of A against rows of B that are read once: memory bound.  Every wave copies whole lines of 32 rows of B (and of
// A, from L2) into a ring of S chunks of its own in LDS, S - 1 of them on their way while one is multiplied; no wave waits for
// another before the end.  (Loading the fragments to registers directly touches every line four times, 32 bytes of 32
// lines per instruction: 3.96 TB/s at one row against 65536 of 4096 amplitudes.)  Pieces lie as in the 128 x 128 tiles.
// AR: rows of A that are copied (8 or 32); those behind the last repeat it.
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
template <int AR, int S> struct ThinPipe {
    static constexpr int kBytes = 4096 + AR * kChunkBytes + 256, kLoads = 4 + AR / 8 + 1;
    uint8_t* ring;
    int lane, r, h;
    uint32_t vb[4], va[AR / 8];
    const uint8_t* scale;        // lanes 0 .. 31: of B's rows, 32 .. 63: of A's

    __device__ __forceinline__ ThinPipe(uint8_t* ring_) : ring(ring_) {
        lane = threadIdx.x & 63;
        r = lane & 31;
        h = lane >> 5;
    }
    __device__ __forceinline__ void rows(const Rows8& A, int64_t row_a, const Rows8& B, int64_t row_b, int64_t cb, int sb) {
        const int la = (int)min((int64_t)32, A.n - row_a) - 1, lb = (int)min((int64_t)32, B.n - row_b) - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = e * 8 + (lane >> 3), piece = (lane & 7) ^ ((row >> 1) & 7);
            vb[e] = (uint32_t)min(row, lb) * (uint32_t)cb + piece * 16;
            if (e < AR / 8) va[e] = (uint32_t)min(row, la) * (uint32_t)cb + piece * 16;
        }
        scale = h ? A.scales + (row_a + min(r, la)) * sb : B.scales + (row_b + min(r, lb)) * sb;
    }
    __device__ __forceinline__ void stage(const uint8_t* a, const uint8_t* b, int c, int slot) {
        uint8_t* to = ring + slot * kBytes;
        const int64_t at = (int64_t)c * kChunkBytes;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            __builtin_amdgcn_global_load_lds((gptr_t)(b + at + (uint64_t)vb[e]), (lptr_t)(to + e * 1024), 16, 0, 0);
#pragma unroll
        for (int e = 0; e < AR / 8; ++e)
            __builtin_amdgcn_global_load_lds((gptr_t)(a + at + (uint64_t)va[e]), (lptr_t)(to + 4096 + e * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((gptr_t)(scale + (c >> 3) * 4), (lptr_t)(to + 4096 + AR * kChunkBytes), 4, 0, 0);
    }
    // SWAP: B's rows are the accumulator's rows (else A's)
    template <bool SWAP> __device__ __forceinline__ void multiply(int c, int slot, v16f& re, v16f& im) {
        const uint8_t* const at = ring + slot * kBytes;
        const int shift = (c >> 1 & 3) * 8, ra = r & (AR - 1);
        const float eb = scale_value((*(const uint32_t*)(at + 4096 + AR * kChunkBytes + r * 4) >> shift) & 255u);
        const float ea = scale_value((*(const uint32_t*)(at + 4096 + AR * kChunkBytes + 128 + r * 4) >> shift) & 255u);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int key = (r >> 1) & 7, keya = (ra >> 1) & 7, pr = 2 * h + s, pi = 4 + 2 * h + s;
            const v4u br = *(const v4u*)(at + r * kChunkBytes + ((pr ^ key) << 4)), bi = *(const v4u*)(at + r * kChunkBytes + ((pi ^ key) << 4));
            const v4u ar = *(const v4u*)(at + 4096 + ra * kChunkBytes + ((pr ^ keya) << 4)), ai = *(const v4u*)(at + 4096 + ra * kChunkBytes + ((pi ^ keya) << 4));
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                v8b xr = widen8(ar[q], ar[q + 1], ea), xi = widen8(ai[q], ai[q + 1], ea);
                v8b yr = widen8(br[q], br[q + 1], eb), yi = widen8(bi[q], bi[q + 1], eb);
                if (SWAP) {
                    const v8b tr = xr, ti = xi;
                    xr = yr; xi = yi; yr = tr; yi = ti;
                }
                re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yr, re, 0, 0, 0);
                im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yi, im, 0, 0, 0);
                re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xi, yi, re, 0, 0, 0);
                im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(negated(xi), yr, im, 0, 0, 0);
            }
        }
    }
    // re, im += over chunks c0 .. c1 - 1 of the rows a, b point at
    template <bool SWAP> __device__ __forceinline__ void run(const uint8_t* a, const uint8_t* b, int c0, int c1, v16f& re, v16f& im) {
#pragma unroll
        for (int k = 0; k < S - 1; ++k)
            if (c0 + k < c1) stage(a, b, c0 + k, k);
        int slot = 0;
        for (int c = c0; c < c1; ++c) {
            const int next = slot ? slot - 1 : S - 1;      // the slot that was read in the round before
            if (c + S - 1 < c1) stage(a, b, c + S - 1, next);
            const int behind = min(S - 1, c1 - 1 - c);     // chunks that may still be on their way
            if (behind == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * kLoads) : "memory");
            else if (behind == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
            else if (behind == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            multiply<SWAP>(c, slot, re, im);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (read before the slot is filled again)
            slot = slot + 1 == S ? 0 : slot + 1;
        }
    }
};
constexpr int kThinLds8 = 4 * 3 * ThinPipe<8, 3>::kBytes, kThinLds32 = 4 * 4 * ThinPipe<32, 4>::kBytes;
static_assert(2 * kThinLds8 <= 160 * 1024 && kThinLds32 <= 160 * 1024 && kThinLds8 >= 4 * 32 * 64 * 4, "LDS");

// K of up to 32 rows (the smaller side of a job, J.A or, if SWAP, J.B) against 32 rows of the other: the four waves split the
// chunks of the item's slice and join their sums in LDS.  One row against 65536 of 4096 amplitudes: 98 us, 5.5 TB/s (the 32 x 32
// tiles of gram8_wave_kernel: 136 us).
template <int AR, bool SWAP> __global__ __launch_bounds__(256) void gram8_thin_kernel(Gram8Args args) {
    constexpr int W = 4, S = AR == 8 ? 3 : 4;
    extern __shared__ uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    ThinPipe<AR, S> pipe(lds + wave * S * ThinPipe<AR, S>::kBytes);
    const int lane = pipe.lane, r = pipe.r;
    const uint32_t item = args.first + blockIdx.x;
    const Gram8JobDev& J = args.job[gram8_job(args, item)];
    uint32_t t, ti, tj;
    int slice;
    gram8_part(J, item - J.begin, t, slice);
    gram8_tile(J, t, ti, tj);
    const Rows8 A = SWAP ? J.B : J.A, B = SWAP ? J.A : J.B;
    const int64_t cb = (int64_t)J.chunks * kChunkBytes, row_a = (int64_t)(SWAP ? tj : ti) * 32, row_b = (int64_t)(SWAP ? ti : tj) * 32;
    v16f re, im;
#pragma unroll
    for (int i = 0; i < 16; ++i) re[i] = im[i] = 0.f;
    const int c0 = max(slice, 0) * J.per, c1 = slice < 0 ? J.chunks : min(J.chunks, c0 + J.per), n = c1 - c0;
    pipe.rows(A, row_a, B, row_b, cb, J.sb);
    pipe.template run<SWAP>(A.codes + row_a * cb, B.codes + row_b * cb, c0 + n * wave / W, c0 + n * (wave + 1) / W, re, im);
    __syncthreads();
    float (*part)[32][64] = (float (*)[32][64])lds;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        part[wave][i][lane] = re[i];
        part[wave][16 + i][lane] = im[i];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16 / W; ++k) {
        const int i = wave * (16 / W) + k;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            x += part[w][i][lane];
            y += part[w][16 + i][lane];
        }
        if (slice < 0) {
            emit(J, (int64_t)ti * 32 + acc_row(lane, i), (int64_t)tj * 32 + r, x, y);
        } else {
            float2* ws = (float2*)(args.ws + J.ws) + ((int64_t)(t - J.whole) * J.slices + slice) * 1024;
            ws[i * 64 + lane] = make_float2(x, y);
        }
    }
}

// ---- 128 x 128 tiles ---------------------------------------------------------------------------------------------------
// Four waves of 64 x 64 (2 x 2 matrix tiles, real and imaginary part: 128 accumulator registers), two workgroups per CU that
// stay and walk the list of tiles.  A step is one chunk of 128 + 128 rows, 32 KiB, copied straight to LDS one step ahead of
// its use (two buffers); the first chunk of the next tile is on its way while a tile is finished, so that rows of a few chunks
// do not pay the latency of memory once per tile.  Row r of a buffer holds its 16-byte piece p at p ^ ((r >> 1) & 7): the 16
// rows that a quarter of a wave reads at once then lie in different banks.
constexpr int kTile = 128;
constexpr int kStage = 2 * kTile * kChunkBytes;
constexpr int kScales = 2 * kStage;                         // a dword of scales (8 chunks) per row, twice
constexpr int kGains = kScales + 2 * 2 * kTile * 4;         // the rows' gains, twice
constexpr int kPipeLds = kGains + 2 * 2 * kTile * 4;

struct TileWork {              // what one pass of the pipeline computes; the same for the whole workgroup
    Rows8 A, B;
    int64_t row_a, row_b;
    int chunks, sb, c0, c1;
};

struct TilePipe {
    uint8_t* lds;
    int wave, lane, r, h;
    const uint8_t* src;        // copies: waves 0 and 1 bring A, 2 and 3 bring B, eight pieces of 8 rows each
    const uint8_t* scale_src;
    uint32_t vo[8], scale_vo;
    int fa, fb, piece[4];
    int buf = 0, area = 0;     // of the step that is computed next
    int next_area = 0;         // of the scales that were copied last

    __device__ __forceinline__ TilePipe(uint8_t* lds_) : lds(lds_) {
        const int tid = threadIdx.x;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        lane = tid & 63;
        r = lane & 31;
        h = lane >> 5;
        // fragments: this lane's row of a 32-row tile, pieces 2 h and 2 h + 1 of either part (which codes of a chunk meet in
        // one instruction is free as long as both operands agree)
        fa = ((wave >> 1) * 64 + r) * kChunkBytes;
        fb = kTile * kChunkBytes + ((wave & 1) * 64 + r) * kChunkBytes;
#pragma unroll
        for (int p = 0; p < 4; ++p) piece[p] = (((p >> 1) * 4 + 2 * h + (p & 1)) ^ ((r >> 1) & 7)) << 4;
    }

    __device__ __forceinline__ void stage(int c, int to_buf, bool first = false) {
        if (first || !(c & 7)) {
            next_area ^= 1;
            asm volatile("" : "+v"(scale_vo));
            __builtin_amdgcn_global_load_lds((gptr_t)(scale_src + (c >> 3) * 4 + (uint64_t)scale_vo),
                                             (lptr_t)(lds + kScales + next_area * 1024 + wave * 256), 4, 0, 0);
        }
        const uint8_t* at = src + (int64_t)c * kChunkBytes;
        uint8_t* to = lds + to_buf * kStage + wave * 8192;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            asm volatile("" : "+v"(vo[e]));      // the sum stays base + 32-bit offset, the instruction's own form
            __builtin_amdgcn_global_load_lds((gptr_t)(at + (uint64_t)vo[e]), (lptr_t)(to + e * 1024), 16, 0, 0);
        }
    }

    // a tile's first chunk, and its gains into half `g` of their area
    __device__ __forceinline__ void open(const TileWork& w, int to_buf, int g) {
        const int64_t cb = (int64_t)w.chunks * kChunkBytes;
        const Rows8 S = wave < 2 ? w.A : w.B;
        const int64_t row0 = wave < 2 ? w.row_a : w.row_b;
        const int last = (int)min((int64_t)kTile, S.n - row0) - 1;      // rows behind the last repeat it
        src = S.codes + row0 * cb;
        scale_src = S.scales + row0 * w.sb;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = (wave & 1) * 64 + e * 8 + (lane >> 3);
            vo[e] = (uint32_t)min(row, last) * (uint32_t)cb + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
        }
        const uint32_t row = (uint32_t)min((wave & 1) * 64 + lane, last);
        scale_vo = row * (uint32_t)w.sb;
        __builtin_amdgcn_global_load_lds((gptr_t)(S.gains + row0 + (uint64_t)row), (lptr_t)(lds + kGains + g * 1024 + wave * 256), 4, 0, 0);
        stage(w.c0, to_buf, true);
    }

    // One step.  STAGE: the copies of the next chunk are issued in its middle, behind the first matrix instructions (12000 rows
    // of 16384 amplitudes, float32 6.6 ms; with the copies first the same within 1 %).
    template <bool STAGE> __device__ __forceinline__ void compute(int c, v16f (&re)[2][2], v16f (&im)[2][2]) {
        const uint8_t* base = lds + buf * kStage;
        const int shift = (c >> 1 & 3) * 8;
        uint32_t sa[2], sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* scale = lds + kScales + area * 1024 + r * 4 + t * 128;
            sa[t] = *(const uint32_t*)(scale + (wave >> 1) * 256);
            sc[t] = *(const uint32_t*)(scale + 512 + (wave & 1) * 256);
        }
        const float ea[2] = {scale_value((sa[0] >> shift) & 255u), scale_value((sa[1] >> shift) & 255u)};
        const float eb[2] = {scale_value((sc[0] >> shift) & 255u), scale_value((sc[1] >> shift) & 255u)};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (STAGE && s == 1) stage(c + 1, buf ^ 1);
            v4u ar[2], ai[2], br[2], bi[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                ar[t] = *(const v4u*)(base + fa + t * 4096 + piece[s]);
                ai[t] = *(const v4u*)(base + fa + t * 4096 + piece[2 + s]);
                br[t] = *(const v4u*)(base + fb + t * 4096 + piece[s]);
                bi[t] = *(const v4u*)(base + fb + t * 4096 + piece[2 + s]);
            }
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                v8b xr[2], xi[2], xn[2], yr[2], yi[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    xr[t] = widen8(ar[t][q], ar[t][q + 1], ea[t]);
                    xi[t] = widen8(ai[t][q], ai[t][q + 1], ea[t]);
                    yr[t] = widen8(br[t][q], br[t][q + 1], eb[t]);
                    yi[t] = widen8(bi[t][q], bi[t][q + 1], eb[t]);
                    xn[t] = negated(xi[t]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        re[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr[i], yr[j], re[i][j], 0, 0, 0);
                        im[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr[i], yi[j], im[i][j], 0, 0, 0);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        re[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xi[i], yi[j], re[i][j], 0, 0, 0);
                        im[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xn[i], yr[j], im[i][j], 0, 0, 0);
                    }
            }
        }
    }

    // Of two workgroups on a CU the matrix unit serves the older one first; left alone, one is through its tile in half the
    // other's time, and the workgroups that share rows in L2 drift apart.  Every 4 steps a wave goes down one level of four and
    // then back to the highest, so the one behind has the higher level most of the time (12000 rows of 16384 amplitudes, float32:
    // 7.27 -> 6.60 ms; 8192 of 4096: 828 -> 797 us; half K 7.25 -> 6.55 ms and 817 -> 790 us).  The level changes before the barrier of a
    // step.
    __device__ __forceinline__ void turn(int c) {
        const int t = (c >> 2) & 3;
        if (t == 0) __builtin_amdgcn_s_setprio(3);
        else if (t == 1) __builtin_amdgcn_s_setprio(2);
        else if (t == 2) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
    }

    // work(k, w): the k-th piece of this workgroup's work, false behind the last.  finish(k, more, gains, room, side, re, im): more: the next
    // one is open; room: 8 KiB of LDS for this wave, the buffer of the last chunk.  STORES: finish issues at least 63 memory
    // instructions.  ASIDE: instead of the next tile's first chunk, aside(k, buffer) fills the free buffer while the last chunk is
    // multiplied, and finish finds it there.
    struct Nothing {
        __device__ void operator()(int, uint8_t*) const {}
    };
    template <bool STORES, bool ASIDE = false, typename Work, typename Finish, typename Aside = Nothing>
    __device__ __forceinline__ void run(Work work, Finish finish, Aside aside = Aside()) {
        TileWork w;
        if (!work(0, w)) return;
        open(w, 0, 0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        for (int k = 0;; ++k) {
            v16f re[2][2], im[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 16; ++q) re[i][j][q] = im[i][j][q] = 0.f;
            int c = w.c0;
            const int c1 = w.c1;
            area = next_area;
            turn(c);
            for (; c + 1 < c1; ++c) {
                compute<true>(c, re, im);
                buf ^= 1;
                if (!((c + 1) & 3)) turn(c + 1);
                __builtin_amdgcn_sched_barrier(0);      // (matrix instructions that sink behind the barrier would not hide it)
                // the copies of the next chunk have landed, and every wave has read the buffer that is filled after it
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                area = (c + 1) & 7 ? area : next_area;
            }
            const bool more = work(k + 1, w);
            if (ASIDE) aside(k, lds + (buf ^ 1) * kStage);
            else if (more) open(w, buf ^ 1, (k + 1) & 1);
            compute<false>(c, re, im);
            if constexpr (ASIDE) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            finish(k, more, (const float*)(lds + kGains + (k & 1) * 1024), lds + buf * kStage + wave * 8192, lds + (buf ^ 1) * kStage, re, im);
            if (!more) return;
            buf ^= 1;
            if constexpr (ASIDE) {
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                open(w, buf, (k + 1) & 1);
            }
            // memory instructions end in order: behind a tile's stores it is enough that all but the youngest 63 have
            if constexpr (STORES) asm volatile("s_waitcnt vmcnt(63) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
    }
};

// Position in a launch -> item: groups of 8 consecutive items (a column of a strip's tiles) are dealt to the eight XCDs in turn, so
// that the 64 tiles of a round on an XCD are 8 columns of one strip; the rest of the list evenly.
__device__ __forceinline__ bool gram8_item(uint32_t total, uint32_t position, uint32_t& item) {
    const uint32_t xcd = position & 7u, seq = position >> 3, full = total >> 6;
    if ((seq >> 3) < full) {
        item = ((((seq >> 3) << 3) + xcd) << 3) + (seq & 7u);
        return true;
    }
    const uint32_t rest = total - (full << 6), share = (rest + 7u) >> 3, in = seq - (full << 3);
    item = (full << 6) + xcd * share + in;
    return in < share && item < total;
}

// Stores through a buffer: the offset -1 is dropped.  The range covers a tile of any row stride the host lets through.
constexpr int kRange = 0x7ffffffe, kRsrc = 0x00027000;
template <typename T> __device__ __forceinline__ void put(T v, __amdgpu_buffer_rsrc_t to, int off, int soff) {
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), to, off, soff, 0);
    else if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), to, off, soff, 0);
    else {
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, v), to, off, soff, 0);
    }
}
// (No scalar offset here: behind a 16-byte buffer store with one the compiler puts no wait state before the next write to its
// data registers, and lanes 12 .. 15 of every 16 were seen to store the new value of the first.)
__device__ __forceinline__ void put16(uint4 v, __amdgpu_buffer_rsrc_t to, int off) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), to, off, 0, 0);
}

// The same in every lane, and known to be: addresses and descriptors made from it stay in scalar registers.
template <typename I> __device__ __forceinline__ I uniform(I v) { return (I)__builtin_amdgcn_readfirstlane((int)v); }

// T: the type of K.  128 x 128 entries per workgroup, 64 x 64 per wave: 128 accumulator registers, two workgroups on a CU, so that one
// multiplies while the other finishes its tile.  Bound by the matrix unit, with the widening between its instructions, at the
// clock that the chip holds under it: 12000 rows of 65536 amplitudes, half K 27.0 ms, 1.40 PFLOP/s; of 16384, half 6.55 ms, float32
// 6.62, float64 6.70, 1.42 (library bf16 product 1.62).  Short rows by what K takes to write: 4096 of 256 amplitudes, half K 24.5 us,
// float32 26.6, float64 42.
template <typename T>
__global__ __launch_bounds__(256, 2) void gram8_tile_kernel(Gram8Args args) {
    extern __shared__ uint8_t lds[];
    TilePipe pipe(lds);
    const int wave = pipe.wave, lane = pipe.lane, r = pipe.r, h = pipe.h;
    struct Where { int job; uint32_t t, ti, tj; int slice; } now{}, before{};      // of the tile that was opened last and the one before
    int round = 0;
    auto item_of = [&](int k, uint32_t& item) {
        // every other round backwards: the list goes from long rows to short ones
        const uint32_t in = k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
        return gram8_item(args.total, in + (uint32_t)k * gridDim.x, item);
    };
    auto work = [&](int k, TileWork& w) {
        uint32_t item;
        round = k;
        if (!item_of(k, item) || item >= args.small) return false;
        before = now;
        Where& p = now;
        p.job = uniform(gram8_job(args, item));
        const Gram8JobDev& J = args.job[p.job];
        gram8_part(J, item - J.begin, p.t, p.slice);
        gram8_tile(J, p.t, p.ti, p.tj);
        p.t = uniform(p.t);
        p.slice = uniform(p.slice);
        p.ti = uniform(p.ti);
        p.tj = uniform(p.tj);
        w.A = J.A;
        w.B = J.B;
        w.row_a = (int64_t)p.ti * kTile;
        w.row_b = (int64_t)p.tj * kTile;
        w.chunks = J.chunks;
        w.sb = J.sb;
        w.c0 = max(p.slice, 0) * J.per;
        w.c1 = p.slice < 0 ? J.chunks : min(J.chunks, w.c0 + J.per);
        return true;
    };
    auto finish = [&](int, bool more, const float* gains, uint8_t* room, const uint8_t* side, v16f (&re)[2][2], v16f (&im)[2][2]) {
        const Where w = more ? before : now, p = {uniform(w.job), uniform(w.t), uniform(w.ti), uniform(w.tj), uniform(w.slice)};
        const Gram8JobDev& J = args.job[p.job];
        if (p.slice >= 0) {
            float2* ws = (float2*)(args.ws + J.ws) + (((int64_t)(p.t - J.whole) * J.slices + p.slice) * 16 + wave * 4) * 1024 + lane;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 16; ++q) ws[(i * 2 + j) * 1024 + q * 64] = make_float2(re[i][j][q], im[i][j][q]);
            return;
        }
        // K from the registers: one of them holds 32 neighbours of two rows.  Entries outside the matrix (symmetric: on or below
        // the diagonal) get an offset that the buffer's range check drops, so the stores have no branches.
        const int S = sizeof(T);
        const bool sym = J.flags & QK_GRAM_SYMMETRIC, diagonal = sym && p.ti == p.tj;
        const int64_t row_t = (int64_t)p.ti * kTile + (wave >> 1) * 64, col_t = (int64_t)p.tj * kTile + (wave & 1) * 64;
        const int rows = (int)min((int64_t)64, J.A.n - row_t), cols = (int)min((int64_t)64, J.B.n - col_t);     // (may be negative)
        const int step = (int)J.ldk * S, ahead = (int)(col_t - row_t);
        const __amdgpu_buffer_rsrc_t K = __builtin_amdgcn_make_buffer_rsrc((char*)J.K + (row_t * J.ldk + col_t) * S, 0, kRange, kRsrc);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = j * 32 + r, off = 4 * h * step + col * S;
                const float gb = gains[kTile + (wave & 1) * 64 + col];
                // rows i * 32 + 4 h + n with n < limit
                int limit = rows - i * 32 - 4 * h;
                if (diagonal) limit = min(limit, col + ahead - i * 32 - 4 * h);
                if (col >= cols) limit = 0;
#pragma unroll
                for (int q = 0; q < 16; q += 4) {
                    const float4 ga = *(const float4*)(gains + (wave >> 1) * 64 + i * 32 + 2 * q + 4 * h);
                    const float g[4] = {ga.x, ga.y, ga.z, ga.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        re[i][j][q + e] = k_value(re[i][j][q + e], im[i][j][q + e], g[e] * gb);
                        const int n = 2 * q + e;
                        put<T>((T)re[i][j][q + e], K, n < limit ? off : -1, (i * 32 + n) * step);
                    }
                }
            }
        if (diagonal && ahead == 0) put<T>((T)1.f, K, lane < min(rows, cols) ? lane * (step + S) : -1, 0);
        T* const mirror = (T*)(sym ? J.K : J.KT);
        if (!mirror) return;
        // The mirror through LDS, [column][its rows], 16-byte pieces of a column at piece ^ key(column); out in whole lines where the
        // rows start on 16 bytes.
        const int64_t ldm = sym ? J.ldk : J.ldkt;
        const int mstep = (int)ldm * S;
        const bool aligned = !(((uintptr_t)mirror | (uint32_t)mstep) & 15), whole = rows >= 64 && cols >= 64 && (!diagonal || ahead > 0);
        if (diagonal && ahead < 0) return;
        const __amdgpu_buffer_rsrc_t M = __builtin_amdgcn_make_buffer_rsrc((char*)mirror + (col_t * ldm + row_t) * S, 0, kRange, kRsrc);
        constexpr int E = 16 / sizeof(T), IP = sizeof(T) == 8 ? 1 : 2, JP = sizeof(T) == 2 ? 2 : 1;      // matrix tiles that 8 KiB hold
        constexpr int RB = IP * 32 * sizeof(T), L = RB / 16;                                             // bytes and pieces of a column
#pragma unroll
        for (int j0 = 0; j0 < 2; j0 += JP)
#pragma unroll
            for (int i0 = 0; i0 < 2; i0 += IP) {
#pragma unroll
                for (int j = 0; j < JP; ++j)
#pragma unroll
                    for (int i = 0; i < IP; ++i)
#pragma unroll
                        for (int q = 0; q < 16; q += 4) {
                            uint8_t* const at = room + (j * 32 + r) * RB;
                            const int key = sizeof(T) == 2 ? (r >> 1) & 7 : r & 15, byte = (i * 32 + 2 * q + 4 * h) * (int)sizeof(T);
                            T u[4] __attribute__((aligned(16)));
#pragma unroll
                            for (int e = 0; e < 4; ++e) u[e] = (T)re[i0 + i][j0 + j][q + e];
                            if constexpr (sizeof(T) == 2) *(uint2*)(at + (((byte >> 4) ^ key) << 4) + (byte & 8)) = *(const uint2*)u;
                            else
#pragma unroll
                                for (int e = 0; e < 4; e += E) *(uint4*)(at + (((byte >> 4) + e / E) ^ key) * 16) = *(const uint4*)(u + e);
                        }
                __builtin_amdgcn_wave_barrier();                // (a wave's LDS accesses stay in order)
                const int s = lane % L, so = j0 * 32 * mstep + i0 * 32 * S;
                // entries of mirror row c that exist: the first ones, up to `limit`
                auto limit_of = [&](int c) {
                    const int col = j0 * 32 + c;
                    int limit = rows;
                    if (diagonal) limit = min(limit, col + ahead);
                    return col < cols ? limit - i0 * 32 : 0;
                };
                if (aligned) {
#pragma unroll 4
                    for (int n = 0; n < JP * L / 2; ++n) {
                        const int c = n * (64 / L) + lane / L, key = sizeof(T) == 2 ? (c >> 1) & 7 : c & 15;
                        const uint4 u = *(const uint4*)(room + c * RB + ((s ^ key) << 4));
                        put16(u, M, whole || (s + 1) * E <= limit_of(c) ? so + c * mstep + s * 16 : -1);
                    }
                    if (!whole) {      // the piece that a row ends in: one lane for each row
                        const int c = lane & (JP * 32 - 1), key = sizeof(T) == 2 ? (c >> 1) & 7 : c & 15;
                        const int limit = lane < JP * 32 ? min(limit_of(c), IP * 32) : 0, last = max(limit, 0) / E;
                        T v[E] __attribute__((aligned(16)));
                        *(uint4*)v = *(const uint4*)(room + c * RB + (((last & (L - 1)) ^ key) << 4));
#pragma unroll
                        for (int e = 0; e < E; ++e) put<T>(v[e], M, last * E + e < limit ? c * mstep + last * 16 + e * S : -1, so);
                    }
                } else {
#pragma unroll 2
                    for (int n = 0; n < JP * L / 2; ++n) {
                        const int c = n * (64 / L) + lane / L, key = sizeof(T) == 2 ? (c >> 1) & 7 : c & 15;
                        T v[E] __attribute__((aligned(16)));
                        *(uint4*)v = *(const uint4*)(room + c * RB + ((s ^ key) << 4));
#pragma unroll
                        for (int e = 0; e < E; ++e) put<T>(v[e], M, s * E + e < limit_of(c) ? c * mstep + s * 16 + e * S : -1, so);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
    };
    pipe.template run<true>(work, finish);
    // the last round in small tiles
    for (uint32_t item; item_of(round, item) && item >= args.small; ++round) {
        const Gram8JobDev& J = args.job[args.n_jobs - 1];
        uint32_t t, ti, tj;
        int slice;
        gram8_part(J, item - J.begin, t, slice);
        gram8_tile(J, t, ti, tj);
        const int64_t row = (int64_t)ti * kTile + (slice >> 2) * 32, col = (int64_t)tj * kTile + (slice & 3) * 32;
        if (row >= J.A.n || col >= J.B.n || ((J.flags & QK_GRAM_SYMMETRIC) && row > col)) continue;
        __syncthreads();
        wave_tile(J, row, col, 0, J.chunks, (float (*)[32][64])lds, nullptr);
    }
}

// Adds the slices of every tile in order and finishes its entries: one thread per entry.  SUB: matrix tiles per tile (1 or 16).
// 140 tiles of 128 x 128 in 3 to 16 slices: 23 us.
template <int SUB>
__global__ __launch_bounds__(256) void gram8_join_kernel(Gram8Args args) {
    const uint32_t tile = blockIdx.x / (4 * SUB);
    uint32_t before = 0;
    int j = 0;
    for (; j + 1 < args.n_jobs; ++j) {
        const uint32_t here = args.job[j].live - args.job[j].whole;
        if (tile < before + here) break;
        before += here;
    }
    const Gram8JobDev& J = args.job[j];
    const uint32_t t = J.whole + (tile - before);
    if (t >= J.live) return;
    uint32_t ti, tj;
    gram8_tile(J, t, ti, tj);
    const int in = (int)(blockIdx.x % (4 * SUB)) * 256 + threadIdx.x, sub = in >> 10, e = in & 1023, lane = e & 63, i = e >> 6;
    const float2* ws = (const float2*)(args.ws + J.ws) + (int64_t)(t - J.whole) * J.slices * SUB * 1024 + in;
    float x = 0.f, y = 0.f;
#pragma unroll 8
    for (int s = 0; s < J.slices; ++s) {
        const float2 v = ws[(int64_t)s * SUB * 1024];
        x += v.x;
        y += v.y;
    }
    // matrix tile of the wave (sub >> 2), then of its 2 x 2
    const int64_t row = SUB == 1 ? (int64_t)ti * 32 : (int64_t)ti * kTile + (sub >> 3) * 64 + ((sub >> 1) & 1) * 32;
    const int64_t col = SUB == 1 ? (int64_t)tj * 32 : (int64_t)tj * kTile + ((sub >> 2) & 1) * 64 + (sub & 1) * 32;
    emit(J, row + acc_row(lane, i), col + (lane & 31), x, y);
}

// ---- decision values -----------------------------------------------------------------------------------------------------
struct Decision8Args {
    Rows8 A, B;
    const float* coef;
    const float* intercept;
    float* out;
    float* ws;             // [parts][C][stride] partial sums
    int64_t ldc, ldo, stride;
    int32_t C, chunks, sb, splits, per, parts;      // per: tile columns of one split; parts: what is left to be joined, 0: out is written at once
};

// The product is taken the other way round (B's rows times A's), so a lane holds 16 of B's rows for ONE row of A: K times the
// coefficients is then a sum over the lane's own registers, and only the two halves of the wave have to be added.  32 rows of A
// (8 with AR = 8) per workgroup against a range of B's.  SPLIT (rows of 8 chunks or more): the four waves share every tile of 32 of
// B's rows, each multiplies a quarter of the chunks and then finishes a quarter of the tile's rows; else every wave has a tile of
// its own (one row against 8192 of 512 amplitudes 8 us shared, 15 each on its own; of 256 the same).  One row against 8192 of 1024 amplitudes (17 MB, 3 us to read): 7.0 us, joining the parts 2.9, 18 from call to call.
template <int AR, bool SPLIT> __global__ __launch_bounds__(256) void decision8_thin_kernel(Decision8Args a) {
    constexpr int W = 4, R = SPLIT ? 16 / W : 16, S = 3;      // R: accumulator registers that a wave finishes
    extern __shared__ uint8_t lds[];
    float* const acc = (float*)(lds + W * S * ThinPipe<AR, S>::kBytes);   // [W][C][32]
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    ThinPipe<AR, S> pipe(lds + wave * S * ThinPipe<AR, S>::kBytes);
    const int lane = pipe.lane, r = pipe.r, h = pipe.h;
    // a wave clears its own sums: no other wave touches them before the barrier behind the tiles
    for (int k = lane; k < 32 * a.C; k += 64) acc[wave * 32 * a.C + k] = 0.f;
    const int64_t row0 = (int64_t)blockIdx.x * AR;
    const int64_t cb = (int64_t)a.chunks * kChunkBytes;
    const float ga = a.A.gains[min(row0 + r, a.A.n - 1)];
    const int tiles = (int)((a.B.n + 31) / 32), t1 = min(tiles, ((int)blockIdx.y + 1) * a.per);
    for (int t = (int)blockIdx.y * a.per + (SPLIT ? 0 : wave); t < t1; t += SPLIT ? 1 : W) {
        const int64_t col0 = (int64_t)t * 32;
        // of this lane's rows of B: gains and the first column's coefficients, on their way while the product is taken
        float gb[R], w[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t col = min(col0 + acc_row(lane, SPLIT ? wave * R + i : i), a.B.n - 1);
            gb[i] = a.B.gains[col];
            w[i] = a.coef[col * a.ldc];
        }
        v16f re, im;
#pragma unroll
        for (int i = 0; i < 16; ++i) re[i] = im[i] = 0.f;
        pipe.rows(a.A, row0, a.B, col0, cb, a.sb);
        pipe.template run<true>(a.A.codes + row0 * cb, a.B.codes + col0 * cb, SPLIT ? a.chunks * wave / W : 0,
                                SPLIT ? a.chunks * (wave + 1) / W : a.chunks, re, im);
        float k[R];
        if constexpr (SPLIT) {
            float (*part)[32][64] = (float (*)[32][64])lds;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                part[wave][i][lane] = re[i];
                part[wave][16 + i][lane] = im[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                float x = 0.f, y = 0.f;
#pragma unroll
                for (int v = 0; v < W; ++v) {
                    x += part[v][wave * R + i][lane];
                    y += part[v][16 + wave * R + i][lane];
                }
                k[i] = x * x + y * y;
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) k[i] = re[i] * re[i] + im[i] * im[i];
        }
#pragma unroll
        for (int i = 0; i < R; ++i) k[i] = col0 + acc_row(lane, SPLIT ? wave * R + i : i) < a.B.n ? k[i] * (ga * gb[i]) : 0.f;
        for (int c = 0; c < a.C; ++c) {
            if (c) {
#pragma unroll
                for (int i = 0; i < R; ++i) w[i] = a.coef[min(col0 + acc_row(lane, SPLIT ? wave * R + i : i), a.B.n - 1) * a.ldc + c];
            }
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i) s += col0 + acc_row(lane, SPLIT ? wave * R + i : i) < a.B.n ? k[i] * w[i] : 0.f;
            s += __shfl_xor(s, 32, 64);
            if (h == 0) acc[(wave * a.C + c) * 32 + r] += s;
        }
    }
    __syncthreads();
    for (int k = tid; k < 32 * a.C; k += 256) {
        const int row = k & 31, c = k >> 5;
        if (row >= AR || row0 + row >= a.A.n) continue;
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < W; ++v) s += acc[v * 32 * a.C + k];
        if (a.parts == 0) a.out[(row0 + row) * a.ldo + c] = s + (a.intercept ? a.intercept[c] : 0.f);
        else a.ws[((int64_t)blockIdx.y * a.C + c) * a.stride + row0 + row] = s;
    }
}

// The same over 128 x 128 tiles: a workgroup keeps 128 rows of A and walks B's tiles of its range.  Each of the two waves that
// share rows of A keeps its own sums of the C columns.
// Up to eight columns (8000 x 4000 rows of 256: five 67 us, eight 70; as MANY 79 and 76): sums in LDS, the coefficients of a wave's 64 rows of B through its part of the free buffer, [column][64]; a
// lane reads four at once, the same for its whole half, and its part of K stays in its registers.
// MANY: out^T += coef^T K^T on FP32 matrix instructions, 32 or 16 columns at a time: a register of K is the right operand as it is.  The
// coefficients of the tile come to the free buffer, [128][C], while the last chunk is multiplied; the sums wait in the workspace
// (which stays in L2), where every lane adds to entries that no other lane touches.
// 16384 x 16384 rows of 1024 amplitudes, one column: 1.46 ms, 1.51 PFLOP/s (library bf16 product 1.39 .. 1.62), bound by the matrix
// unit with the widening between its instructions.  3001 x 10007 rows of 256, 45 columns: 113 us; a tile takes 10 us for K and
// 12 for its columns, 6 of them FP32 matrix instructions.
constexpr int kLdsColumns = 8;
constexpr int kDecisionLds = kPipeLds + 2 * kLdsColumns * kTile * 4;
static_assert(2 * kDecisionLds <= 160 * 1024, "two workgroups per CU");
static_assert(QK_DECISION8_MAX_C * kTile * 4 <= kStage, "a tile's coefficients fit a buffer");

template <bool MANY> __global__ __launch_bounds__(256, 2) void decision8_tile_kernel(Decision8Args a) {
    extern __shared__ uint8_t lds[];
    TilePipe pipe(lds);
    const int tid = threadIdx.x, wave = pipe.wave, lane = pipe.lane, r = pipe.r, h = pipe.h;
    const int xs = (wave & 1) * 64, ys = (wave >> 1) * 64;
    const int64_t row0 = (int64_t)blockIdx.x * kTile, mp = (int64_t)gridDim.x * kTile;
    float* const sums = (float*)(lds + kPipeLds);
    const int tiles = (int)((a.B.n + kTile - 1) / kTile), t0 = (int)blockIdx.y * a.per, t1 = min(tiles, t0 + a.per);
    auto work = [&](int k, TileWork& w) {
        if (t0 + k >= t1) return false;
        w.A = a.B;
        w.B = a.A;
        w.row_a = (int64_t)(t0 + k) * kTile;
        w.row_b = row0;
        w.chunks = a.chunks;
        w.sb = a.sb;
        w.c0 = 0;
        w.c1 = a.chunks;
        return true;
    };
    // re <- K of this wave's 64 x 64, 0 behind B's last row
    auto kernel = [&](int k, const float* gains, v16f (&re)[2][2], v16f (&im)[2][2]) {
        const float gx[2] = {gains[kTile + xs + r], gains[kTile + xs + 32 + r]};
        const int left = (int)min((int64_t)64, a.B.n - (int64_t)(t0 + k) * kTile - ys) - 4 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
                const float4 gy = *(const float4*)(gains + ys + i * 32 + 2 * q + 4 * h);
                const float g[4] = {gy.x, gy.y, gy.z, gy.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float v = (re[i][j][q + e] * re[i][j][q + e] + im[i][j][q + e] * im[i][j][q + e]) * (gx[j] * g[e]);
                        re[i][j][q + e] = i * 32 + 2 * q + e < left ? v : 0.f;
                    }
            }
    };
    if constexpr (MANY) {
        auto aside = [&](int k, uint8_t* to) {
            // element n of the tile's [128][C]: rows behind the last repeat it
            const int64_t y0 = (int64_t)(t0 + k) * kTile;
            const int last = (int)min((int64_t)kTile, a.B.n - y0) - 1, total = kTile * a.C, dr = 256 / a.C, dc = 256 - dr * a.C;
            int row = tid / a.C, c = tid - row * a.C;
            for (int n = 0; n < total; n += 256) {      // (the last round may run over: the buffer has the room, the row is repeated)
                __builtin_amdgcn_global_load_lds((gptr_t)(a.coef + (y0 + min(row, last)) * a.ldc + c), (lptr_t)(to + n * 4 + wave * 256), 4, 0, 0);
                row += dr;
                c += dc;
                if (c >= a.C) {
                    c -= a.C;
                    ++row;
                }
            }
        };
        auto finish = [&](int k, bool, const float* gains, uint8_t*, const uint8_t* side, v16f (&re)[2][2], v16f (&im)[2][2]) {
            kernel(k, gains, re, im);
            const int left = (int)min((int64_t)64, a.B.n - (int64_t)(t0 + k) * kTile - ys) - 4 * h;
            int c0 = 0;
            for (; a.C - c0 > 16; c0 += 32) {
                const int n = a.C - c0 - 4 * h;
                float* const at = a.ws + (((int64_t)blockIdx.y * 2 + (wave >> 1)) * a.C + c0 + 4 * h) * mp + row0 + xs + r;
                float old[2][16];
                v16f sum[2];
#pragma unroll
                for (int q = 0; q < 16; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int c = 8 * (q >> 2) + (q & 3);
                        old[j][q] = 0.f;
                        if (k && c < n) old[j][q] = at[c * mp + j * 32];
                        sum[j][q] = 0.f;
                    }
                const float* const coef = (const float*)side + min(c0 + r, a.C - 1) + (ys + 4 * h) * a.C;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        const int row = i * 32 + 8 * (q >> 2) + (q & 3);
                        const float v = coef[row * a.C], w = row < left ? v : 0.f;
#pragma unroll
                        for (int j = 0; j < 2; ++j) sum[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(w, re[i][j][q], sum[j], 0, 0, 0);
                    }
#pragma unroll
                for (int q = 0; q < 16; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int c = 8 * (q >> 2) + (q & 3);
                        if (c < n) at[c * mp + j * 32] = old[j][q] + sum[j][q];
                    }
            }
            // 16 or fewer are left: four 16 x 16 products at once, two for the rows of either half of the wave, in half the time
            // (3001 x 10007 rows of 256: 45 columns 119 -> 113 us, 16 columns 83 -> 80)
            if (c0 < a.C) {
                const int g = lane >> 4, x = lane & 15, n = a.C - c0 - 4 * g;
                float* const at = a.ws + (((int64_t)blockIdx.y * 2 + (wave >> 1)) * a.C + c0 + 4 * g) * mp + row0 + xs + x;
                float old[2][8];
                v16f sum[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        if (q < 8) {
                            old[j][q] = 0.f;
                            if (k && (q & 3) < n) old[j][q] = at[(q & 3) * mp + j * 32 + 16 * (q >> 2)];
                        }
                        sum[j][q] = 0.f;
                    }
                const float* const coef = (const float*)side + min(c0 + x, a.C - 1) + (ys + 4 * h) * a.C;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        const int row = i * 32 + 8 * (q >> 2) + (q & 3);
                        const float v = coef[row * a.C], w = row < left ? v : 0.f;
#pragma unroll
                        for (int j = 0; j < 2; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x1f32(w, re[i][j][q], sum[j], 0, 0, 0);
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if ((q & 3) < n) at[(q & 3) * mp + j * 32 + 16 * (q >> 2)] = old[j][q] + (sum[j][q] + sum[j][q + 8]);
            }
        };
        pipe.run<false, true>(work, finish, aside);
    } else {
        auto finish = [&](int k, bool, const float* gains, uint8_t* room, const uint8_t*, v16f (&re)[2][2], v16f (&im)[2][2]) {
            float* const coef = (float*)room;
            // (0 behind B's last row: K is 0 there, and an infinite coefficient must not meet it)
            const int64_t at = (int64_t)(t0 + k) * kTile + ys + lane, y = min(at, a.B.n - 1);
#pragma unroll 4
            for (int c = 0; c < a.C; ++c) {
                const float v = a.coef[y * a.ldc + c];
                coef[c * 64 + lane] = at == y ? v : 0.f;
            }
            kernel(k, gains, re, im);
            __builtin_amdgcn_wave_barrier();
            for (int c = 0; c < a.C; ++c) {
                float s[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 16; q += 4) {
                        const float4 w = *(const float4*)(coef + c * 64 + i * 32 + 2 * q + 4 * h);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            s[j] += re[i][j][q] * w.x + re[i][j][q + 1] * w.y + re[i][j][q + 2] * w.z + re[i][j][q + 3] * w.w;
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) s[j] += __shfl_xor(s[j], 32, 64);
                float* const to = sums + ((wave >> 1) * kLdsColumns + c) * kTile + xs + lane;
                const float mine = h ? s[1] : s[0];                  // lane half h keeps the rows of matrix tile j = h
                *to = k ? *to + mine : mine;
            }
            __builtin_amdgcn_wave_barrier();
        };
        pipe.run<false>(work, finish);
        __syncthreads();
        for (int k = tid; k < kTile * a.C; k += 256) {
            const int row = k & (kTile - 1), c = k >> 7;
            if (row0 + row >= a.A.n) continue;
            const float s = sums[c * kTile + row] + sums[(kLdsColumns + c) * kTile + row];
            if (a.parts == 0) a.out[(row0 + row) * a.ldo + c] = s + (a.intercept ? a.intercept[c] : 0.f);
            else a.ws[((int64_t)blockIdx.y * a.C + c) * mp + row0 + row] = s;
        }
    }
}

// Adds the parts, ws[part][C][stride], in a fixed order: 16 rows per workgroup, each by 16 threads that take every 16th part.
// parts == 0: only the intercept.
__global__ __launch_bounds__(256) void decision8_join_kernel(Decision8Args a) {
    __shared__ double sum[16][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.y;
    for (int64_t row0 = (int64_t)blockIdx.x * 16; row0 < a.A.n; row0 += (int64_t)gridDim.x * 16) {
        const int64_t row = row0 + x;
        double s = 0.0;
        if (row < a.A.n) {
#pragma unroll 4
            for (int p = y; p < a.parts; p += 16) s += (double)a.ws[((int64_t)p * a.C + c) * a.stride + row];
        }
        sum[y][x] = s;
        __syncthreads();
        if (y == 0 && row < a.A.n) {
            s = a.intercept ? (double)a.intercept[c] : 0.0;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += sum[k][x];
            a.out[row * a.ldo + c] = (float)s;
        }
        __syncthreads();
    }
}

// out = K coef + intercept for a K that is there: one workgroup per entry.
__global__ __launch_bounds__(256) void decision8_rows_kernel(Decision8Args a) {
    __shared__ double sum[4];
    const int64_t row = blockIdx.x;
    const int c = blockIdx.y;
    const float* const K = a.ws + row * a.B.n;
    double s = 0.0;
#pragma unroll 4
    for (int64_t j = threadIdx.x; j < a.B.n; j += 256) s += (double)K[j] * (double)a.coef[j * a.ldc + c];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.out[row * a.ldo + c] = (float)(sum[0] + sum[1] + sum[2] + sum[3] + (a.intercept ? (double)a.intercept[c] : 0.0));
}

// ---- host side -------------------------------------------------------------------------------------------------------------
namespace {
constexpr int64_t kMaxD = (int64_t)1 << 26;

int check_states(const char* who, const qk_states8& s) {
    if (s.rows < 0) return fail(QK_ERR_INVALID, std::string(who) + ": negative row count");
    if (s.rows > 0x7fffffffLL) return fail(QK_ERR_UNSUPPORTED, std::string(who) + ": more than 2^31 - 1 rows");
    if (s.rows && (!s.codes || !s.scales || !s.gains)) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer in a store");
    if (((uintptr_t)s.codes & 15) || ((uintptr_t)s.scales & 3) || ((uintptr_t)s.gains & 3))
        return fail(QK_ERR_INVALID, std::string(who) + ": codes need 16-byte alignment, scales and gains 4");
    return QK_OK;
}
int check_dim(const char* who, int64_t D) {
    if (D < 1 || D > kMaxD) return fail(QK_ERR_INVALID, std::string(who) + ": D must be in 1..2^26");
    return QK_OK;
}

Rows8 rows8(const qk_states8& s) { return Rows8{(const uint8_t*)s.codes, (const uint8_t*)s.scales, s.gains, s.rows}; }

// Which kernel takes a job.  The 128 x 128 kernel reads every row from L2 once for 128 others and needs enough tiles, or tile
// steps, to fill the chip; the 32 x 32 kernel starts at once, takes few rows without waste and spreads a small job over more
// workgroups.  Measured, us with 32 x 32 / 128 x 128: float32, 61 tiles of 512 amplitudes 18.2 / 18.0, of 1024 25.9 / 27.7; 120 of 512
// 25.1 / 18.8; 15 of 4096 (977 steps) 27.2 / 27.8, 34 of 4096 (2197) 56 / 35.  float16: 63 of 512 13.7 / 17.7, 90 of 512 18.5 / 17.8, 120 of 512
// 23.0 / 17.9, 15 of 4096 26.3 / 25.1, 35 of 4096 57 / 34.
// The kernels for few rows copy 8 or 32 of them beside every 32 of the others: 32 x 32 tiles / these, one row against 65536 of
// 512 amplitudes 18.5 / 19.4, of 1024 28.2 / 28.2, of 4096 136 / 98; nine rows against 64 MB of 2048 18.5 / 20.0, of 4096 26.2 / 16.6, against
// 16 MB 12.4 / 13.0.
enum Gram8Kind { GK_WAVE, GK_THIN8, GK_THIN32, GK_THIN8_SWAP, GK_THIN32_SWAP, GK_TILE, GK_TILE_F64, GK_TILE_F16, GK_KINDS };
constexpr double g_tiles = 96, g_steps = 1024;
std::atomic<int> g_path{0};      // development hook: 0 by rule, 1 always 32 x 32, 2 always 128 x 128, 3 the kernels for few rows where they can

int64_t live_tiles(const qk_gram8_job& j, int64_t tile) {
    const int64_t tm = (j.A.rows + tile - 1) / tile, tn = (j.B.rows + tile - 1) / tile;
    return (j.flags & QK_GRAM_SYMMETRIC) ? tm * (tm + 1) / 2 : tm * tn;
}

// 128 x 128 tiles that a job fills (its parts of tiles added up); 0: too few rows, or rows so long or so far apart that 32 bits
// do not hold the offsets inside a tile
double tiles_of(const qk_gram8_job& j) {
    const int64_t m = std::min(j.A.rows, j.B.rows), n = std::max(j.A.rows, j.B.rows);
    if (m < (g_path.load(std::memory_order_relaxed) == 2 ? 1 : 33) || code_bytes(j.D) > (int64_t)1 << 24) return 0;
    if (std::max(j.ldk, j.KT ? j.ldkt : 0) * 8 > (int64_t)1 << 23) return 0;
    return (double)std::max<int64_t>(m, 64) * (double)n / (kTile * kTile) * (j.flags & QK_GRAM_SYMMETRIC ? 0.5 : 1.0);
}

// tiles, steps (tiles times chunks): of all jobs of the call
Gram8Kind kind_of(const qk_gram8_job& j, double tiles, double steps) {
    const int path = g_path.load(std::memory_order_relaxed);
    // up to 8 rows against more than 2 MiB of codes in rows of 16 chunks or more, or 32 against 16 MiB in rows of 64: memory bound
    const int64_t few = std::min(j.A.rows, j.B.rows), many = std::max(j.A.rows, j.B.rows);
    if (!(j.flags & QK_GRAM_SYMMETRIC) && few <= 32 && code_bytes(j.D) <= (int64_t)1 << 26 &&
        (path == 3 || (path == 0 && j.D > (few <= 8 ? 960 : 4032) && many * code_bytes(j.D) > (int64_t)1 << (few <= 8 ? 21 : 24)))) {
        const bool swap = j.B.rows < j.A.rows;
        return few <= 8 ? (swap ? GK_THIN8_SWAP : GK_THIN8) : (swap ? GK_THIN32_SWAP : GK_THIN32);
    }
    if (path == 1 || path == 3 || tiles_of(j) == 0 || (path == 0 && tiles < g_tiles && steps < g_steps)) return GK_WAVE;
    return j.flags & QK_GRAM8_F16 ? GK_TILE_F16 : j.flags & QK_GRAM8_F64 ? GK_TILE_F64 : GK_TILE;
}

// One launch's worth of jobs of one kind: tiles, slices, workspace.
struct Gram8Plan {
    Gram8Args args;
    uint32_t join_tiles;
    size_t ws_floats;
};

// Workgroups that run at a time
constexpr int64_t slots(Gram8Kind kind) { return kind == GK_WAVE ? 1024 : kind == GK_THIN32 || kind == GK_THIN32_SWAP ? 256 : 512; }

// Which of a job's tiles are cut into slices of their rows, and into how many: those of the last round over the chip's slots,
// where cutting brings more than it costs.  Measured for 128 x 128 tiles: a step (a chunk of a tile) takes 3.0 us with two workgroups on
// every CU, 1.45 to 1.6 with one; another round 4 us more; joining a launch, 0.085 us per
// tile and 0.01 per slice (64 tiles in two slices 13 us, in eight 14, 121 in two 16).  32 x 32 tiles: 0.4 us a step, 5 us and
// the slices' way out and back at 5 TB/s.  behind: steps of the jobs behind this one that fill up the round.  second: the call's
// last tiles are in the second round.
void cut(Gram8Kind kind, int64_t live, int chunks, int64_t taken, double behind, bool second, Gram8JobDev& d) {
    const int64_t all = slots(kind), side = kind < GK_TILE ? 32 : kTile, last = (taken + live) % all, tail = std::min(live, last);
    const double pair = 3.0, one = 1.55;
    auto cost = [&](int n, int per) {
        const int64_t items = tail * n, rounds = (items + all - 1) / all;
        if (kind < GK_TILE) return (double)(rounds * per) * 0.4 + (n > 1 ? 5.0 + (double)(items * side * side * 16) / 5e6 : 0.0);
        const double step = behind == 0 && 2 * items <= all ? one : pair * (rounds > 1 ? 1.0 : 0.67 + 0.33 * (double)items / (double)all);
        return (double)rounds * (per * step + 4.0) + (n > 1 ? 6.0 + 0.085 * (double)tail + 0.01 * (double)items : 0.0);
    };
    d.whole = (uint32_t)live;
    d.slices = 1;
    d.small = 0;
    d.per = chunks;
    if (tail == 0 || behind >= 0.5 * (double)((all - last) * chunks)) return;      // the jobs behind it fill the round
    double best = cost(1, chunks);
    const int most = std::min(kind < GK_TILE ? chunks / 16 : chunks / 4, 256);
    for (int n = 2; n <= most; ++n) {
        const int per = (chunks + n - 1) / n;
        if ((chunks + per - 1) / per != n) continue;
        const double here = cost(n, per);
        if (here < best) {
            best = here;
            d.slices = n;
            d.per = per;
            d.whole = (uint32_t)(live - tail);
        }
    }
    // Few tiles of short rows behind one full round: as 32 x 32 tiles they take one step of every workgroup.  (4096 rows of 256
    // amplitudes, 528 tiles: half K 34.4 -> 24.2 us, float32 35.7 -> 26.7, float64 59 -> 42; 49 tiles over, half: rows of 64 21.2 -> 21.6,
    // of 256 34.6 -> 32.1; 83 tiles over 22.2 -> 25.6 and 35.3 -> 37.1.)
    if (second && kind >= GK_TILE && d.slices == 1 && chunks <= 8 && last <= live && 16 * tail <= all) {
        d.small = 1;
        d.slices = 16;
        d.whole = (uint32_t)(live - tail);
    }
}

int plan_gram8(const qk_gram8_job* jobs, const int* which, int n, Gram8Kind kind, Gram8Plan& p) {
    std::memset(&p, 0, sizeof(p));
    const int64_t side = kind < GK_TILE ? 32 : kTile;
    int64_t items = 0;
    p.args.small = 0xffffffffu;
    for (int k = 0; k < n; ++k) {
        const qk_gram8_job& j = jobs[which[k]];
        Gram8JobDev& d = p.args.job[p.args.n_jobs++];
        d.A = rows8(j.A);
        d.B = rows8(j.B);
        d.K = j.K;
        d.KT = j.KT;
        d.ldk = j.ldk;
        d.ldkt = j.ldkt;
        d.flags = j.flags;
        d.chunks = (int32_t)((j.D + kChunk - 1) / kChunk);
        d.sb = (int32_t)scale_bytes(j.D);
        d.tiles_m = (int32_t)((j.A.rows + side - 1) / side);
        d.tiles_n = (int32_t)((j.B.rows + side - 1) / side);
        const int64_t live = live_tiles(j, side);
        // what the jobs behind this one (shorter rows) bring to the slots that its last tiles leave free in their round, in steps
        double behind = 0;
        const int64_t taken = items % slots(kind);
        int64_t room = slots(kind) - (taken + live) % slots(kind);
        for (int l = k + 1; l < n && room; ++l) {
            const int64_t some = std::min(room, live_tiles(jobs[which[l]], side));
            behind += (double)some * (double)((jobs[which[l]].D + kChunk - 1) / kChunk);
            room -= some;
        }
        cut(kind, live, d.chunks, taken, behind, k == n - 1 && items + live > slots(kind) && items + live < 2 * slots(kind), d);
        if (items + live * d.slices > 0x7fffffffLL) return fail(QK_ERR_UNSUPPORTED, "qk_gram8_jobs_dev: too many tiles; split the call");
        d.live = (uint32_t)live;
        d.begin = (uint32_t)items;
        items += d.whole + (live - d.whole) * d.slices;
        if (d.small) p.args.small = d.begin + d.whole;
        else if (d.whole < live) {
            d.ws = (int64_t)p.ws_floats;
            p.ws_floats += (size_t)(live - d.whole) * d.slices * 2 * side * side;
            p.join_tiles += (uint32_t)(live - d.whole);
        }
    }
    p.args.total = (uint32_t)items;
    return QK_OK;
}

// The launches of a call, in order: `each(plan, kind)`.  Jobs with long rows go first, so that a launch does not end on them.
template <typename F> int gram8_launches(const qk_gram8_job* jobs, int n, F each) {
    std::vector<int> by[GK_KINDS];
    double tiles = 0, steps = 0;
    for (int k = 0; k < n; ++k) {
        const double t = tiles_of(jobs[k]);
        tiles += t;
        steps += t * (double)((jobs[k].D + kChunk - 1) / kChunk);
    }
    for (int k = 0; k < n; ++k)
        if (jobs[k].A.rows && jobs[k].B.rows) by[kind_of(jobs[k], tiles, steps)].push_back(k);
    for (int kind = GK_KINDS - 1; kind >= 0; --kind) {
        std::stable_sort(by[kind].begin(), by[kind].end(), [&](int a, int b) { return jobs[a].D > jobs[b].D; });
        for (size_t k = 0; k < by[kind].size(); k += kGram8Jobs) {
            Gram8Plan p;
            int rc = plan_gram8(jobs, by[kind].data() + k, (int)std::min<size_t>(kGram8Jobs, by[kind].size() - k), (Gram8Kind)kind, p);
            if (rc || (rc = each(p, (Gram8Kind)kind))) return rc;
        }
    }
    return QK_OK;
}

int check_gram8(const qk_gram8_job* jobs, int n) {
    const char* who = "qk_gram8_jobs_dev";
    if (n < 0 || (n && !jobs)) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer or negative count");
    for (int k = 0; k < n; ++k) {
        const qk_gram8_job& j = jobs[k];
        int rc;
        if ((rc = check_dim(who, j.D)) || (rc = check_states(who, j.A)) || (rc = check_states(who, j.B))) return rc;
        if ((j.flags & QK_GRAM8_F16) && (j.flags & QK_GRAM8_F64)) return fail(QK_ERR_INVALID, std::string(who) + ": K has one type");
        if (j.flags & ~(QK_GRAM_SYMMETRIC | QK_GRAM8_F16 | QK_GRAM8_F64)) return fail(QK_ERR_INVALID, std::string(who) + ": unknown flag");
        if ((j.flags & QK_GRAM_SYMMETRIC) && (j.A.codes != j.B.codes || j.A.scales != j.B.scales || j.A.gains != j.B.gains ||
                                              j.A.rows != j.B.rows))
            return fail(QK_ERR_INVALID, std::string(who) + ": a symmetric job needs the same store on both sides");
        if (!j.A.rows || !j.B.rows) continue;
        if (!j.K) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer in job");
        if ((j.flags & QK_GRAM_SYMMETRIC) && j.KT) return fail(QK_ERR_INVALID, std::string(who) + ": a symmetric job writes its mirror into K");
        if (j.ldk < j.B.rows || (j.KT && j.ldkt < j.A.rows))
            return fail(QK_ERR_INVALID, std::string(who) + ": leading dimension smaller than the block");
    }
    return QK_OK;
}

// -> whether the 128 x 128 kernel takes it
// (us in 32-row tiles / in 128 x 128 ones, whose rows are not cut: 24 of them of 4096 amplitudes 31 / 94, 61 of 1024 24.0 / 28.3, of 4096
// 53 / 95, 95 of 1024 38 / 29, of 4096 90 / 93, 120 of 1024 39 / 29; of 256 and less the same)
bool plan_decision8(int64_t M, int64_t N, int64_t D, int C, Decision8Args& a) {
    a.C = C;
    a.chunks = (int32_t)((D + kChunk - 1) / kChunk);
    a.sb = (int32_t)scale_bytes(D);
    const int path = g_path.load(std::memory_order_relaxed);
    const double area = (double)std::max<int64_t>(M, 64) * (double)std::max<int64_t>(N, 64) / (kTile * kTile);
    const bool tile = code_bytes(D) <= (int64_t)1 << 24 &&
                      (path == 2 || (path == 0 && M > 32 && area >= g_tiles));
    const int64_t side = tile ? kTile : M <= 8 ? 8 : 32, tm = (M + side - 1) / side, tn = (N + (tile ? kTile : 32) - 1) / (tile ? kTile : 32);
    const int64_t want = tile ? std::max<int64_t>(1, std::min<int64_t>(tn, 512 / std::max<int64_t>(tm, 1)))
                              : std::max<int64_t>(1, std::min<int64_t>(a.chunks >= 8 ? tn : (tn + 3) / 4, 1024 / std::max<int64_t>(tm, 1)));
    a.per = (int32_t)std::max<int64_t>(1, (tn + want - 1) / want);
    a.splits = (int32_t)std::max<int64_t>(1, (tn + a.per - 1) / a.per);
    a.stride = tm * side;
    a.parts = tile && C > kLdsColumns ? 2 * a.splits : a.splits > 1 ? a.splits : 0;
    return tile;
}

// A few rows against few long ones: the 32-row tiles would be less than one for every other CU, each with a long way to go, so K
// goes through memory, its rows cut by gram8's rule.  (Tiles / this, us: one row against 1000 of 9000 amplitudes 25 / 14, of 65536 132 / 32;
// 32 rows against 1000 of 65536 154 / 36; one against 4000 of 9000 25.4 / 25.5, 8000 of 9000 29 / 37.)  Its ends hold for the rows they
// were measured on: behind them the tiles walk whole rows of 65536 amplitudes too -- 33 rows against 1000 take 156 us (gram8 68), one
// against 4097 174 (gram8 128), 128 against 12288 1.59 ms (gram8 0.70).
bool decision8_by_rows(int64_t M, int64_t N, int64_t D) {
    return g_path.load(std::memory_order_relaxed) == 0 && M <= 32 && D > 64 * kChunk && N <= 4096;
}
qk_gram8_job decision8_job(const qk_states8& x, const qk_states8& y, int64_t D, void* K) {
    qk_gram8_job j;
    std::memset(&j, 0, sizeof(j));
    j.A = x;
    j.B = y;
    j.D = D;
    j.K = K;
    j.ldk = y.rows;
    return j;
}
// An entry point that plans on the heap: no exception leaves the library.
template <typename F> int no_throw(const char* who, F body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(QK_ERR_INVALID, std::string(who) + ": out of memory on the host");
    }
}

size_t decision8_k_bytes(int64_t M, int64_t N) { return (size_t)((M * N * (int64_t)sizeof(float) + 255) & ~(int64_t)255); }
}  // namespace
}  // namespace qk

using namespace qk;

extern "C" int qk_states8_layout(int64_t D, int64_t* code_row_bytes, int64_t* scale_row_bytes) {
    const int rc = check_dim("qk_states8_layout", D);
    if (rc) return rc;
    if (!code_row_bytes || !scale_row_bytes) return fail(QK_ERR_INVALID, "qk_states8_layout: null pointer");
    *code_row_bytes = code_bytes(D);
    *scale_row_bytes = scale_bytes(D);
    return QK_OK;
}

extern "C" int qk_states8_write_dev(const void* psi, int f32, int64_t ldpsi, int64_t D, const qk_states8* to, void* stream) {
    const char* who = "qk_states8_write_dev";
    if (!to) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    int rc;
    if ((rc = check_dim(who, D)) || (rc = check_states(who, *to))) return rc;
    const int64_t N = to->rows;
    if (N == 0) return QK_OK;
    if (!psi) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    if (ldpsi < D) return fail(QK_ERR_INVALID, std::string(who) + ": row stride smaller than D");
    if ((uintptr_t)psi & (f32 ? 7 : 15)) return fail(QK_ERR_INVALID, std::string(who) + ": states need the alignment of their type");
    const int64_t blocks = (D + kBlock - 1) / kBlock;
    uint8_t *codes = (uint8_t*)to->codes, *scales = (uint8_t*)to->scales;
    float* gains = (float*)to->gains;
    const hipStream_t s = (hipStream_t)stream;
    // A wave takes two blocks at a time: one wave per row up to 8 blocks, four up to 32, else sixteen.  (complex64, 512 MB: 1024
    // amplitudes 94 us with one wave, 106 with four; 2048 102 and 89; 8192 96 with four, 90 with sixteen; 16384 99 and 92.)
    const int wpr = blocks <= 8 ? 1 : blocks <= 32 ? 4 : 16;
    const int rows = wpr == 1 ? 4 : 1, threads = wpr == 16 ? 1024 : 256;      // of a workgroup
    const int64_t most = kThreads / threads * rows, cb = code_bytes(D), sb = scale_bytes(D);
#define QK_WRITE8(T, W)                                                                                                       \
    hipLaunchKernelGGL((states8_write_kernel<T, W>), dim3((unsigned)((n + rows - 1) / rows)), dim3(threads), 0, s,            \
                       (const char*)psi + first * ldpsi * (f32 ? 8 : 16), n, D, ldpsi, codes + first * cb, scales + first * sb, gains + first)
    for (int64_t first = 0; first < N; first += most) {
        const int64_t n = std::min(most, N - first);
        if (f32) {
            if (wpr == 1) QK_WRITE8(float, 1); else if (wpr == 4) QK_WRITE8(float, 4); else QK_WRITE8(float, 16);
        } else {
            if (wpr == 1) QK_WRITE8(double, 1); else if (wpr == 4) QK_WRITE8(double, 4); else QK_WRITE8(double, 16);
        }
    }
#undef QK_WRITE8
    QK_HIP(hipGetLastError());
    return QK_OK;
}

extern "C" int qk_states8_read_dev(const qk_states8* from, int64_t D, const int64_t* index, int64_t N, void* psi, int f32,
                                   int64_t ldpsi, void* stream) {
    const char* who = "qk_states8_read_dev";
    if (!from) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    int rc;
    if ((rc = check_dim(who, D)) || (rc = check_states(who, *from))) return rc;
    if (N < 0 || N > 0x7fffffffLL) return fail(QK_ERR_INVALID, std::string(who) + ": row count out of range");
    if (N == 0) return QK_OK;
    if (!psi) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    if (!index && N > from->rows) return fail(QK_ERR_INVALID, std::string(who) + ": more rows than the store holds");
    if (ldpsi < D) return fail(QK_ERR_INVALID, std::string(who) + ": row stride smaller than D");
    if ((uintptr_t)psi & (f32 ? 7 : 15)) return fail(QK_ERR_INVALID, std::string(who) + ": states need the alignment of their type");
    const bool longer = D >= 512;
    const int64_t rows = std::max<int64_t>(1, kReadPairs / ((D + 1) / 2)), segments = (D + 511) / 512;
    const int64_t grid = longer ? (N * segments + 3) / 4 : (N + rows - 1) / rows;
    if (grid > kThreads / 256) return fail(QK_ERR_UNSUPPORTED, std::string(who) + ": too many amplitudes; split the call");
    const uint8_t *codes = (const uint8_t*)from->codes, *scales = (const uint8_t*)from->scales;
    const bool vec = !((uintptr_t)psi & 15) && (ldpsi * (f32 ? 8 : 16)) % 16 == 0;
    const dim3 g((unsigned)grid), b(256);
    const hipStream_t s = (hipStream_t)stream;
#define QK_READ8(T, VEC)                                                                                                             \
    if (longer)                                                                                                                      \
        hipLaunchKernelGGL((states8_read_long_kernel<T, VEC>), g, b, 0, s, codes, scales, index, from->rows, (uint32_t)(N * segments), D, \
                           psi, ldpsi, (uint32_t)segments);                                                                          \
    else                                                                                                                             \
        hipLaunchKernelGGL((states8_read_kernel<T, VEC>), g, b, 0, s, codes, scales, index, from->rows, N, D, psi, ldpsi, (uint32_t)rows)
    if (!f32) { QK_READ8(double, true); }
    else if (vec) { QK_READ8(float, true); }
    else { QK_READ8(float, false); }
#undef QK_READ8
    QK_HIP(hipGetLastError());
    return QK_OK;
}

namespace {
int gram8_workspace(const qk_gram8_job* jobs, int n_jobs, size_t* bytes) {
    if (!bytes) return fail(QK_ERR_INVALID, "qk_gram8_workspace: null pointer");
    *bytes = 0;
    const int rc = check_gram8(jobs, n_jobs);
    if (rc) return rc;
    return gram8_launches(jobs, n_jobs, [&](const Gram8Plan& p, Gram8Kind) {
        *bytes = std::max(*bytes, p.ws_floats * sizeof(float));      // the launches of a call use it one after the other
        return QK_OK;
    });
}
}  // namespace
extern "C" int qk_gram8_workspace(const qk_gram8_job* jobs, int n_jobs, size_t* bytes) {
    return no_throw("qk_gram8_workspace", [&] { return gram8_workspace(jobs, n_jobs, bytes); });
}

// A launch with more LDS than a kernel may have unasked
template <typename K, typename A> int launch8(K kernel, dim3 grid, int lds, hipStream_t s, const A& args, DeviceOnce& once, int most) {
    if (once.pending()) {
        QK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, most));
        once.done();
    }
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, args);
    QK_HIP(hipGetLastError());
    return QK_OK;
}
#define QK_TILE8(T)                                                                                                  \
    do {                                                                                                             \
        static DeviceOnce once;                                                                                      \
        const int rc8 = launch8(gram8_tile_kernel<T>, dealt, kPipeLds, s, p.args, once, kPipeLds);                   \
        if (rc8) return rc8;                                                                                         \
    } while (0)
#define QK_THIN8(AR, SWAP)                                                                                           \
    do {                                                                                                             \
        static DeviceOnce once;                                                                                      \
        constexpr int lds8 = AR == 8 ? kThinLds8 : kThinLds32;                                                       \
        const int rc8 = launch8(gram8_thin_kernel<AR, SWAP>, some, lds8, s, p.args, once, lds8);                     \
        if (rc8) return rc8;                                                                                         \
    } while (0)

namespace {
int gram8_jobs_dev(const qk_gram8_job* jobs, int n_jobs, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_gram8(jobs, n_jobs);
    if (rc) return rc;
    if ((uintptr_t)ws & 15) return fail(QK_ERR_INVALID, "qk_gram8_jobs_dev: the workspace needs 16-byte alignment");
    rc = gram8_launches(jobs, n_jobs, [&](const Gram8Plan& p, Gram8Kind) {      // all of it is checked before any of it runs
        if (p.ws_floats * sizeof(float) > ws_bytes || (p.ws_floats && !ws))
            return fail(QK_ERR_INVALID, "qk_gram8_jobs_dev: workspace smaller than qk_gram8_workspace asks for");
        return (int)QK_OK;
    });
    if (rc) return rc;
    const hipStream_t s = (hipStream_t)stream;
    return gram8_launches(jobs, n_jobs, [&](Gram8Plan& p, Gram8Kind kind) {
        p.args.ws = (float*)ws;
        const uint32_t total = p.args.total, full = total >> 6;
        // two workgroups per CU that stay (one for each item: 5000 x 7001 rows of 64 amplitudes, half K 39 against 36 us, float32 43 against 40;
        // rows of 256 and more within 2 %); where the last round is of small tiles, one for each item: those start wherever one ends (4096 rows
        // of 256 amplitudes, float32 30.6 -> 28.0 us)
        const dim3 dealt(std::min<uint32_t>(p.args.small < total ? 0x7fffffffu : 512u, (full << 6) + 8 * ((total - (full << 6) + 7) >> 3)));
        const uint32_t most = (uint32_t)(kThreads / 256);
        if (kind < GK_TILE)
            for (; p.args.first < total; p.args.first += most) {
                const dim3 some(std::min(most, total - p.args.first));
                if (kind == GK_WAVE) hipLaunchKernelGGL(gram8_wave_kernel, some, dim3(256), 0, s, p.args);
                else if (kind == GK_THIN8) QK_THIN8(8, false);
                else if (kind == GK_THIN8_SWAP) QK_THIN8(8, true);
                else if (kind == GK_THIN32) QK_THIN8(32, false);
                else QK_THIN8(32, true);
            }
        else if (kind == GK_TILE) QK_TILE8(float);
        else if (kind == GK_TILE_F64) QK_TILE8(double);
        else QK_TILE8(_Float16);
        QK_HIP(hipGetLastError());
        if (p.join_tiles) {
            if (kind < GK_TILE) hipLaunchKernelGGL(gram8_join_kernel<1>, dim3(p.join_tiles * 4), dim3(256), 0, s, p.args);
            else hipLaunchKernelGGL(gram8_join_kernel<16>, dim3(p.join_tiles * 64), dim3(256), 0, s, p.args);
            QK_HIP(hipGetLastError());
        }
        return (int)QK_OK;
    });
}
}  // namespace
extern "C" int qk_gram8_jobs_dev(const qk_gram8_job* jobs, int n_jobs, void* ws, size_t ws_bytes, void* stream) {
    return no_throw("qk_gram8_jobs_dev", [&] { return gram8_jobs_dev(jobs, n_jobs, ws, ws_bytes, stream); });
}

// Development hook (not in the public header): which kernel the products of 8-bit stores use, whatever the rule says.
extern "C" int qk_gram8_set_path(const char* name) {
    const std::string s = name ? name : "";
    if (s == "auto") g_path = 0;
    else if (s == "wave") g_path = 1;
    else if (s == "tile") g_path = 2;
    else if (s == "thin") g_path = 3;
    else return fail(QK_ERR_INVALID, "qk_gram8_set_path: auto, wave, tile or thin");
    return QK_OK;
}

namespace {
int decision8_workspace(int64_t M, int64_t N, int64_t D, int C, size_t* bytes) {
    const char* who = "qk_decision8_workspace";
    if (!bytes) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    *bytes = 0;
    int rc;
    if ((rc = check_dim(who, D))) return rc;
    if (M < 0 || N < 0 || M > 0x7fffffffLL || N > 0x7fffffffLL) return fail(QK_ERR_INVALID, std::string(who) + ": row count out of range");
    if (C < 1 || C > QK_DECISION8_MAX_C) return fail(QK_ERR_UNSUPPORTED, std::string(who) + ": 1 to QK_DECISION8_MAX_C columns");
    if (M == 0 || N == 0) return QK_OK;
    Decision8Args a;
    std::memset(&a, 0, sizeof(a));
    if (decision8_by_rows(M, N, D)) {
        const qk_gram8_job job = decision8_job({nullptr, nullptr, nullptr, M}, {nullptr, nullptr, nullptr, N}, D, nullptr);
        size_t gram = 0;
        rc = gram8_launches(&job, 1, [&](const Gram8Plan& p, Gram8Kind) {
            gram = std::max(gram, p.ws_floats * sizeof(float));
            return (int)QK_OK;
        });
        *bytes = decision8_k_bytes(M, N) + gram;
        return rc;
    }
    plan_decision8(M, N, D, C, a);
    *bytes = (size_t)a.parts * C * a.stride * sizeof(float);
    return QK_OK;
}

int decision8_dev(const qk_states8* x, const qk_states8* y, int64_t D, const float* coef, int64_t ldc, int C, const float* intercept,
                  float* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "qk_decision8_dev";
    if (!x || !y) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    int rc;
    if ((rc = check_dim(who, D)) || (rc = check_states(who, *x)) || (rc = check_states(who, *y))) return rc;
    size_t need = 0;
    if ((rc = decision8_workspace(x->rows, y->rows, D, C, &need))) return rc;
    if (x->rows == 0) return QK_OK;
    if (!out || (y->rows && !coef)) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    if (ldc < C || ldo < C) return fail(QK_ERR_INVALID, std::string(who) + ": row stride smaller than C");
    if (need > ws_bytes || (need && !ws)) return fail(QK_ERR_INVALID, std::string(who) + ": workspace smaller than qk_decision8_workspace asks for");
    if ((uintptr_t)ws & 15) return fail(QK_ERR_INVALID, std::string(who) + ": the workspace needs 16-byte alignment");
    Decision8Args a;
    std::memset(&a, 0, sizeof(a));
    a.A = rows8(*x);
    a.B = rows8(*y);
    a.coef = coef;
    a.intercept = intercept;
    a.out = out;
    a.ws = (float*)ws;
    a.ldc = ldc;
    a.ldo = ldo;
    const bool tile = plan_decision8(x->rows, y->rows, D, C, a);
    const hipStream_t s = (hipStream_t)stream;
    const dim3 joins((unsigned)std::min<int64_t>((x->rows + 15) / 16, 1 << 20), (unsigned)C);
    if (y->rows == 0) {
        a.parts = 0;
        hipLaunchKernelGGL(decision8_join_kernel, joins, dim3(256), 0, s, a);
        QK_HIP(hipGetLastError());
        return QK_OK;
    }
    if (decision8_by_rows(x->rows, y->rows, D)) {
        const size_t k = decision8_k_bytes(x->rows, y->rows);
        const qk_gram8_job job = decision8_job(*x, *y, D, ws);
        if ((rc = gram8_jobs_dev(&job, 1, (char*)ws + k, ws_bytes - k, stream))) return rc;
        hipLaunchKernelGGL(decision8_rows_kernel, dim3((unsigned)x->rows, (unsigned)C), dim3(256), 0, s, a);
        QK_HIP(hipGetLastError());
        return QK_OK;
    }
    if (tile) {
        static DeviceOnce once[2];
        const dim3 grid((unsigned)((x->rows + kTile - 1) / kTile), (unsigned)a.splits);
        rc = C > kLdsColumns ? launch8(decision8_tile_kernel<true>, grid, kPipeLds, s, a, once[0], kPipeLds)
                             : launch8(decision8_tile_kernel<false>, grid, kDecisionLds, s, a, once[1], kDecisionLds);
    } else {
        const int side = x->rows <= 8 ? 8 : 32, sums = 4 * 32 * C * (int)sizeof(float);
        constexpr int most = 4 * 32 * QK_DECISION8_MAX_C * (int)sizeof(float), ring8 = 4 * 3 * ThinPipe<8, 3>::kBytes, ring32 = 4 * 3 * ThinPipe<32, 3>::kBytes;
        static_assert(ring32 + most <= 160 * 1024, "LDS");
        const dim3 grid((unsigned)((x->rows + side - 1) / side), (unsigned)a.splits);
        static DeviceOnce once[4];
        if (side == 8)
            rc = a.chunks >= 8 ? launch8(decision8_thin_kernel<8, true>, grid, ring8 + sums, s, a, once[0], ring8 + most)
                               : launch8(decision8_thin_kernel<8, false>, grid, ring8 + sums, s, a, once[1], ring8 + most);
        else
            rc = a.chunks >= 8 ? launch8(decision8_thin_kernel<32, true>, grid, ring32 + sums, s, a, once[2], ring32 + most)
                               : launch8(decision8_thin_kernel<32, false>, grid, ring32 + sums, s, a, once[3], ring32 + most);
    }
    if (rc) return rc;
    if (a.parts) {
        hipLaunchKernelGGL(decision8_join_kernel, joins, dim3(256), 0, s, a);
        QK_HIP(hipGetLastError());
    }
    return QK_OK;
}
}  // namespace

extern "C" int qk_decision8_workspace(int64_t M, int64_t N, int64_t D, int C, size_t* bytes) {
    return no_throw("qk_decision8_workspace", [&] { return decision8_workspace(M, N, D, C, bytes); });
}

extern "C" int qk_decision8_dev(const qk_states8* x, const qk_states8* y, int64_t D, const float* coef, int64_t ldc, int C,
                                const float* intercept, float* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    return no_throw("qk_decision8_dev", [&] { return decision8_dev(x, y, D, coef, ldc, C, intercept, out, ldo, ws, ws_bytes, stream); });
}
