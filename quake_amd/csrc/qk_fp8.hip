// 8-bit state stores and the products over them (gfx950): e4m3 codes with one power-of-two scale for each block of 128
// amplitudes.
//
//   write     psi -> codes, scales, gains            code = e4m3(component * 2^-e), e = the least integer with
//                                                    max |component of the block| * 2^-e <= 448
//   read      codes, scales -> code * 2^e
//   gram8     K_ij = gain_i gain_j |sum_b conj(q_i[b]) q_j[b]|^2,  gain = ||psi||^2 / ||q||^2
//   decision8 out[m][c] = sum_j K_mj coef[j][c] + intercept[c], K never written
//
// A row of D amplitudes is laid out as chunks of 64 amplitudes: 64 real codes, then 64 imaginary codes (128 bytes, one
// cache line); the last chunk is padded with zero codes.  Two chunks share one scale byte e + 127.  Scales are powers of
// two because that is exact: multiplying by one never rounds, and an e4m3 code has the same relative step whatever the
// scale (the scale only keeps the block inside the format's 2^18 range).
//
// Arithmetic of the products: codes are widened to bf16 (exact: e4m3 has 4 significant bits, bf16 has 8 and FP32's
// exponents) with the block's scale applied in the same instruction, products and sums are FP32 on the matrix cores.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "qk_common.h"

namespace qk {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;            // amplitudes per chunk
constexpr int kChunkBytes = 128;
constexpr int kBlock = 128;           // amplitudes per scale
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

// One half-wave (32 lanes) holds one block: lane i has amplitudes i, i + 32, i + 64, i + 96 (coalesced loads).  WPR waves
// work on one row and its sums meet in LDS.
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
        for (int64_t b0 = 2 * sub; b0 < sb; b0 += 2 * WPR) {
            const int64_t b = b0 + half;
            float re[4], im[4], top = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t at = b * kBlock + 32 * k + i;
                P v;
                v.x = v.y = 0;
                if (at < D) v = src[at];
                norm += (double)v.x * (double)v.x + (double)v.y * (double)v.y;
                re[k] = to_f32_odd(v.x);
                im[k] = to_f32_odd(v.y);
                top = fmaxf(top, fmaxf(fabsf(re[k]), fabsf(im[k])));      // (fmax drops NaN)
            }
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 32));
            const int e = scale_exponent(top);
            uint32_t wr = 0, wi = 0;      // byte k: the code of amplitude 32 k + i
            float sq = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = ldexpf(re[k], -e), c = ldexpf(im[k], -e);
                uint32_t p = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, c, 0, false) & 0xffffu;
                p &= ~(((p & 0x7f7fu) + 0x0101u) & 0x8080u);      // one code for NaN: 0x7f
                wr |= (p & 0xffu) << (8 * k);
                wi |= ((p >> 8) & 0xffu) << (8 * k);
                const float qa = __builtin_amdgcn_cvt_f32_fp8((int)p, 0), qc = __builtin_amdgcn_cvt_f32_fp8((int)p, 1);
                sq += qa * qa + qc * qc;
            }
            kept += ldexp((double)sq, 2 * e);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t at = b * kBlock + 32 * k + i;
                const int64_t o = (at >> 6) * kChunkBytes + (at & 63);
                if (o < cb) {
                    dst[o] = (uint8_t)(wr >> (8 * k));
                    dst[o + kChunk] = (uint8_t)(wi >> (8 * k));
                }
            }
            if (i == 0 && b < sb) sc[b] = (uint8_t)(b < blocks ? e + 127 : 127);
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
// Two amplitudes per thread.  A row number outside 0 .. of - 1 gives a row of NaN.
template <typename T>
__global__ __launch_bounds__(256) void states8_read_kernel(const uint8_t* codes, const uint8_t* scales, const int64_t* index,
                                                           int64_t of, int64_t N, int64_t D, void* out_, int64_t ldo) {
    typedef typename Pair<T>::type P;
    const int64_t cb = (D + kChunk - 1) / kChunk * kChunkBytes, sb = ((D + kBlock - 1) / kBlock + 3) / 4 * 4;
    const int64_t per = (D + 1) / 2;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < N * per; t += (int64_t)gridDim.x * 256) {
        const int64_t n = t / per, at = 2 * (t - n * per);
        const int64_t row = index ? index[n] : n;
        P* out = (P*)out_ + n * ldo + at;
        P v[2];
        if (row < 0 || row >= of) {
            v[0].x = v[0].y = v[1].x = v[1].y = (T)__builtin_nanf("");
        } else {
            const uint8_t* c = codes + row * cb + (at >> 6) * kChunkBytes + (at & 63);
            const int e = (int)scales[row * sb + (at >> 7)] - 127;
            const int r = *(const uint16_t*)c, s = *(const uint16_t*)(c + kChunk);
            v[0].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r, 0), e);
            v[1].x = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(r, 1), e);
            v[0].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s, 0), e);
            v[1].y = (T)ldexpf(__builtin_amdgcn_cvt_f32_fp8(s, 1), e);
        }
        out[0] = v[0];
        if (at + 1 < D) out[1] = v[1];
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
    int32_t tiles_n;           // tile columns
    int32_t slices;            // the row's chunks are cut into this many slices of `per` chunks
    int32_t per;
    uint32_t live;             // tiles that have to be computed
    uint32_t begin;            // items (tile x slice) of the jobs before
};

struct Gram8Args {
    Gram8JobDev job[kGram8Jobs];
    int32_t n_jobs;
    uint32_t total;            // items
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

// One entry of K and its mirror (symmetric: the entries below the diagonal are the ones above it, so K is symmetric to the
// bit; summed on their own they would differ in the order of the imaginary part's two halves).
__device__ __forceinline__ void emit(const Gram8JobDev& J, int64_t row, int64_t col, float re, float im) {
    const bool sym = J.flags & QK_GRAM_SYMMETRIC;
    if (row >= J.A.n || col >= J.B.n || (sym && row > col)) return;
    float k = (re * re + im * im) * (J.A.gains[row] * J.B.gains[col]);
    if (sym && row == col) k = 1.f;
    store_k(J.K, row * J.ldk + col, k, J.flags);
    if (sym && row != col) store_k(J.K, col * J.ldk + row, k, J.flags);
    if (J.KT) store_k(J.KT, col * J.ldkt + row, k, J.flags);
}

// Tile t of a job: row-major over the tiles that have to be computed (symmetric: those on or above the diagonal).
__device__ __forceinline__ void gram8_tile(const Gram8JobDev& J, uint32_t t, uint32_t& ti, uint32_t& tj) {
    const uint32_t T = (uint32_t)J.tiles_n;
    if (!(J.flags & QK_GRAM_SYMMETRIC)) {
        ti = t / T;
        tj = t - ti * T;
        return;
    }
    uint32_t lo = 0, hi = T - 1;             // the last row whose first tile is at or before t
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if ((uint64_t)mid * T - (uint64_t)mid * (mid - 1) / 2 <= t) lo = mid; else hi = mid - 1;
    }
    ti = lo;
    tj = lo + (t - (uint32_t)((uint64_t)lo * T - (uint64_t)lo * (lo - 1) / 2));
}

__device__ __forceinline__ int gram8_job(const Gram8Args& a, uint32_t item) {
    int j = 0;
    while (j + 1 < a.n_jobs && a.job[j + 1].begin <= item) ++j;
    return j;
}

// re += conj(a) c, im of the same, over chunks c0, c0 + step, ... < c1 of two 32-row operands (pa, pb: this lane's rows,
// offset by its half).  The matrix instruction sums 8 codes of either half of the wave; which 8 is free as long as both
// operands agree, so a lane takes whole 16-byte pieces.
__device__ __forceinline__ void wave_product(const uint8_t* pa, const uint8_t* sa, const uint8_t* pb, const uint8_t* sb, int c0,
                                             int c1, int step, v16f& re, v16f& im) {
    for (int c = c0; c < c1; c += step) {
        const float fa = scale_value(sa[c >> 1]), fb = scale_value(sb[c >> 1]);
        const uint8_t *a = pa + (int64_t)c * kChunkBytes, *b = pb + (int64_t)c * kChunkBytes;
        v4u ar[2], ai[2], br[2], bi[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            ar[s] = *(const v4u*)(a + 32 * s);
            ai[s] = *(const v4u*)(a + 64 + 32 * s);
            br[s] = *(const v4u*)(b + 32 * s);
            bi[s] = *(const v4u*)(b + 64 + 32 * s);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                const v8b xr = widen8(ar[s][q], ar[s][q + 1], fa), xi = widen8(ai[s][q], ai[s][q + 1], fa);
                const v8b yr = widen8(br[s][q], br[s][q + 1], fb), yi = widen8(bi[s][q], bi[s][q + 1], fb);
                re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yr, re, 0, 0, 0);
                re = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xi, yi, re, 0, 0, 0);
                im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xr, yi, im, 0, 0, 0);
                im = __builtin_amdgcn_mfma_f32_32x32x16_bf16(negated(xi), yr, im, 0, 0, 0);
            }
    }
}

// A 32 x 32 tile per workgroup, the chunks of its slice dealt to four waves, their sums joined in LDS.
__global__ __launch_bounds__(256) void gram8_wave_kernel(Gram8Args args) {
    constexpr int W = 4;
    __shared__ float part[W][32][64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const uint32_t item = blockIdx.x;
    const Gram8JobDev& J = args.job[gram8_job(args, item)];
    const uint32_t in = item - J.begin, slice = in / J.live, t = in - slice * J.live;
    uint32_t ti, tj;
    gram8_tile(J, t, ti, tj);
    const int64_t cb = (int64_t)J.chunks * kChunkBytes;
    const int64_t ra = min((int64_t)ti * 32 + r, J.A.n - 1), rb = min((int64_t)tj * 32 + r, J.B.n - 1);
    v16f re, im;
#pragma unroll
    for (int i = 0; i < 16; ++i) re[i] = im[i] = 0.f;
    const int c0 = (int)slice * J.per, c1 = min(J.chunks, c0 + J.per);
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
        if (J.slices == 1) {
            emit(J, (int64_t)ti * 32 + acc_row(lane, i), (int64_t)tj * 32 + r, x, y);
        } else {
            float2* ws = (float2*)(args.ws + J.ws) + ((int64_t)t * J.slices + slice) * 1024;
            ws[i * 64 + lane] = make_float2(x, y);
        }
    }
}

// Adds the slices of every tile in order and finishes its entries: one thread per entry, four workgroups per tile.
__global__ __launch_bounds__(256) void gram8_join_kernel(Gram8Args args) {
    const uint32_t tile = blockIdx.x >> 2;
    uint32_t before = 0;
    int j = 0;
    for (; j + 1 < args.n_jobs; ++j) {
        const uint32_t here = args.job[j].slices > 1 ? args.job[j].live : 0;
        if (tile < before + here) break;
        before += here;
    }
    const Gram8JobDev& J = args.job[j];
    const uint32_t t = tile - before;
    if (J.slices <= 1 || t >= J.live) return;
    uint32_t ti, tj;
    gram8_tile(J, t, ti, tj);
    const int e = (blockIdx.x & 3) * 256 + threadIdx.x, lane = e & 63, i = e >> 6;
    const float2* ws = (const float2*)(args.ws + J.ws) + (int64_t)t * J.slices * 1024 + e;
    float x = 0.f, y = 0.f;
    for (int s = 0; s < J.slices; ++s) {
        const float2 v = ws[(int64_t)s * 1024];
        x += v.x;
        y += v.y;
    }
    emit(J, (int64_t)ti * 32 + acc_row(lane, i), (int64_t)tj * 32 + (lane & 31), x, y);
}

// ---- decision values -----------------------------------------------------------------------------------------------------
struct Decision8Args {
    Rows8 A, B;
    const float* coef;
    const float* intercept;
    float* out;
    float* ws;             // splits x M x C partial sums when splits > 1
    int64_t ldc, ldo;
    int32_t C, chunks, sb, splits, per;      // per: tile columns of one split
};

// Sum of v[0..15] over the 32 lanes of a half; lane gets the sum of register `row_of(lane)`: halving exchanges, so every
// step moves half of what is left.
__device__ __forceinline__ float half_reduce(float* v, int lane) {
#pragma unroll
    for (int step = 0; step < 4; ++step) {
        const int m = 16 >> step, n = 8 >> step;
        const bool up = lane & m;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) {
                const float send = up ? v[k] : v[k + n], keep = up ? v[k + n] : v[k];
                v[k] = keep + __shfl_xor(send, m, 64);
            }
    }
    return v[0] + __shfl_xor(v[0], 1, 64);
}
__device__ __forceinline__ int half_reduce_register(int lane) { return (lane >> 1) & 15; }

// 32 rows of A against a range of B's rows: each of four waves takes every fourth tile of 32 of them, turns its K tile into
// C partial sums per row at once and adds them up in LDS.
__global__ __launch_bounds__(256) void decision8_wave_kernel(Decision8Args a) {
    constexpr int W = 4;
    extern __shared__ float acc[];            // [W][32][C]
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 31, h = lane >> 5;
    for (int k = tid; k < W * 32 * a.C; k += 256) acc[k] = 0.f;
    __syncthreads();
    const int64_t row0 = (int64_t)blockIdx.x * 32;
    const int64_t cb = (int64_t)a.chunks * kChunkBytes, ra = min(row0 + r, a.A.n - 1);
    float ga[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) ga[i] = a.A.gains[min(row0 + acc_row(lane, i), a.A.n - 1)];
    const int tiles = (int)((a.B.n + 31) / 32), t1 = min(tiles, ((int)blockIdx.y + 1) * a.per);
    for (int t = (int)blockIdx.y * a.per + wave; t < t1; t += W) {
        const int64_t col = (int64_t)t * 32 + r, rb = min(col, a.B.n - 1);
        v16f re, im;
#pragma unroll
        for (int i = 0; i < 16; ++i) re[i] = im[i] = 0.f;
        wave_product(a.A.codes + ra * cb + 16 * h, a.A.scales + ra * a.sb, a.B.codes + rb * cb + 16 * h, a.B.scales + rb * a.sb, 0, a.chunks,
                     1, re, im);
        const float gb = a.B.gains[rb];
        float k[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) k[i] = (re[i] * re[i] + im[i] * im[i]) * (ga[i] * gb);
        for (int c = 0; c < a.C; ++c) {
            const float w = col < a.B.n ? a.coef[col * a.ldc + c] : 0.f;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = col < a.B.n ? k[i] * w : 0.f;
            const float s = half_reduce(v, lane);
            if (!(lane & 1)) acc[(wave * 32 + acc_row(lane, half_reduce_register(lane))) * a.C + c] += s;
        }
    }
    __syncthreads();
    for (int k = tid; k < 32 * a.C; k += 256) {
        const int row = k / a.C, c = k - row * a.C;
        if (row0 + row >= a.A.n) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += acc[w * 32 * a.C + k];
        if (a.splits == 1) a.out[(row0 + row) * a.ldo + c] = s + (a.intercept ? a.intercept[c] : 0.f);
        else a.ws[((int64_t)blockIdx.y * a.A.n + row0 + row) * a.C + c] = s;
    }
}

__global__ __launch_bounds__(256) void decision8_join_kernel(Decision8Args a) {
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k >= a.A.n * a.C) return;
    const int64_t row = k / a.C;
    const int c = (int)(k - row * a.C);
    double s = 0.0;
    for (int p = 0; p < a.splits; ++p) s += (double)a.ws[(int64_t)p * a.A.n * a.C + k];
    a.out[row * a.ldo + c] = (float)(s + (a.intercept ? (double)a.intercept[c] : 0.0));
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

// One launch's worth of jobs: tiles, slices, workspace.
struct Gram8Plan {
    Gram8Args args;
    uint32_t join_tiles;
    size_t ws_floats;
};

int plan_gram8(const qk_gram8_job* jobs, int n, Gram8Plan& p) {
    std::memset(&p, 0, sizeof(p));
    int64_t tiles = 0;
    for (int k = 0; k < n; ++k) {
        const qk_gram8_job& j = jobs[k];
        const int64_t tm = (j.A.rows + 31) / 32, tn = (j.B.rows + 31) / 32;
        tiles += (j.flags & QK_GRAM_SYMMETRIC) ? tm * (tm + 1) / 2 : tm * tn;
    }
    int64_t items = 0;
    for (int k = 0; k < n; ++k) {
        const qk_gram8_job& j = jobs[k];
        if (!j.A.rows || !j.B.rows) continue;
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
        const int64_t tm = (j.A.rows + 31) / 32, tn = (j.B.rows + 31) / 32;
        d.tiles_n = (int32_t)tn;
        const int64_t live = (j.flags & QK_GRAM_SYMMETRIC) ? tm * (tm + 1) / 2 : tm * tn;
        // few tiles with long rows: slices of at least 16 chunks (four for each wave), enough for about 1024 workgroups
        int64_t slices = std::max<int64_t>(1, std::min<int64_t>(d.chunks / 16, 1024 / std::max<int64_t>(tiles, 1)));
        d.per = (int32_t)((d.chunks + slices - 1) / slices);
        d.slices = (d.chunks + d.per - 1) / d.per;
        if (items + live * d.slices > 0x7fffffffLL) return fail(QK_ERR_UNSUPPORTED, "qk_gram8_jobs_dev: too many tiles; split the call");
        d.live = (uint32_t)live;
        d.begin = (uint32_t)items;
        items += live * d.slices;
        if (d.slices > 1) {
            d.ws = (int64_t)p.ws_floats;
            p.ws_floats += (size_t)live * d.slices * 2048;
            p.join_tiles += (uint32_t)live;
        }
    }
    p.args.total = (uint32_t)items;
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

int plan_decision8(int64_t M, int64_t N, int64_t D, int C, Decision8Args& a) {
    a.C = C;
    a.chunks = (int32_t)((D + kChunk - 1) / kChunk);
    a.sb = (int32_t)scale_bytes(D);
    const int64_t tm = (M + 31) / 32, tn = (N + 31) / 32;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>((tn + 3) / 4, 1024 / std::max<int64_t>(tm, 1)));
    a.per = (int32_t)std::max<int64_t>(1, (tn + want - 1) / want);
    a.splits = (int32_t)std::max<int64_t>(1, (tn + a.per - 1) / a.per);
    return QK_OK;
}
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
    // a wave takes two blocks at a time: one wave per row up to 8 blocks, sixteen for the longest rows
    const int wpr = blocks <= 8 ? 1 : blocks <= 64 ? 4 : 16;
    const int64_t grid = wpr == 1 ? (N + 3) / 4 : N;
    if (grid > 0x7fffffffLL) return fail(QK_ERR_UNSUPPORTED, std::string(who) + ": too many rows");
#define QK_WRITE8(T, W) \
    hipLaunchKernelGGL((states8_write_kernel<T, W>), dim3((unsigned)grid), dim3(W < 4 ? 256 : 64 * W), 0, s, psi, N, D, ldpsi, codes, scales, gains)
    if (f32) {
        if (wpr == 1) QK_WRITE8(float, 1); else if (wpr == 4) QK_WRITE8(float, 4); else QK_WRITE8(float, 16);
    } else {
        if (wpr == 1) QK_WRITE8(double, 1); else if (wpr == 4) QK_WRITE8(double, 4); else QK_WRITE8(double, 16);
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
    const int64_t work = N * ((D + 1) / 2);
    const unsigned grid = (unsigned)std::min<int64_t>((work + 255) / 256, 1 << 20);
    const uint8_t *codes = (const uint8_t*)from->codes, *scales = (const uint8_t*)from->scales;
    if (f32)
        hipLaunchKernelGGL(states8_read_kernel<float>, dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, scales, index, from->rows, N, D, psi, ldpsi);
    else
        hipLaunchKernelGGL(states8_read_kernel<double>, dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, scales, index, from->rows, N, D, psi, ldpsi);
    QK_HIP(hipGetLastError());
    return QK_OK;
}

extern "C" int qk_gram8_workspace(const qk_gram8_job* jobs, int n_jobs, size_t* bytes) {
    if (!bytes) return fail(QK_ERR_INVALID, "qk_gram8_workspace: null pointer");
    *bytes = 0;
    int rc = check_gram8(jobs, n_jobs);
    if (rc) return rc;
    size_t most = 0;
    for (int k = 0; k < n_jobs; k += kGram8Jobs) {
        Gram8Plan p;
        if ((rc = plan_gram8(jobs + k, std::min(kGram8Jobs, n_jobs - k), p))) return rc;
        most = std::max(most, p.ws_floats * sizeof(float));
    }
    *bytes = most;
    return QK_OK;
}

extern "C" int qk_gram8_jobs_dev(const qk_gram8_job* jobs, int n_jobs, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_gram8(jobs, n_jobs);
    if (rc) return rc;
    for (int k = 0; k < n_jobs; k += kGram8Jobs) {
        Gram8Plan p;
        if ((rc = plan_gram8(jobs + k, std::min(kGram8Jobs, n_jobs - k), p))) return rc;
        if (p.args.n_jobs == 0) continue;
        if (p.ws_floats * sizeof(float) > ws_bytes || (p.ws_floats && !ws))
            return fail(QK_ERR_INVALID, "qk_gram8_jobs_dev: workspace smaller than qk_gram8_workspace asks for");
        if ((uintptr_t)ws & 15) return fail(QK_ERR_INVALID, "qk_gram8_jobs_dev: the workspace needs 16-byte alignment");
        p.args.ws = (float*)ws;
        hipLaunchKernelGGL(gram8_wave_kernel, dim3(p.args.total), dim3(256), 0, (hipStream_t)stream, p.args);
        QK_HIP(hipGetLastError());
        if (p.join_tiles) {
            hipLaunchKernelGGL(gram8_join_kernel, dim3(p.join_tiles * 4), dim3(256), 0, (hipStream_t)stream, p.args);
            QK_HIP(hipGetLastError());
        }
    }
    return QK_OK;
}

extern "C" int qk_decision8_workspace(int64_t M, int64_t N, int64_t D, int C, size_t* bytes) {
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
    plan_decision8(M, N, D, C, a);
    if (a.splits > 1) *bytes = (size_t)a.splits * M * C * sizeof(float);
    return QK_OK;
}

extern "C" int qk_decision8_dev(const qk_states8* x, const qk_states8* y, int64_t D, const float* coef, int64_t ldc, int C,
                                const float* intercept, float* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "qk_decision8_dev";
    if (!x || !y) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    int rc;
    if ((rc = check_dim(who, D)) || (rc = check_states(who, *x)) || (rc = check_states(who, *y))) return rc;
    size_t need = 0;
    if ((rc = qk_decision8_workspace(x->rows, y->rows, D, C, &need))) return rc;
    if (x->rows == 0) return QK_OK;
    if (!out || (y->rows && !coef)) return fail(QK_ERR_INVALID, std::string(who) + ": null pointer");
    if (ldc < C || ldo < C) return fail(QK_ERR_INVALID, std::string(who) + ": row stride smaller than C");
    if (need > ws_bytes || (need && !ws)) return fail(QK_ERR_INVALID, std::string(who) + ": workspace smaller than qk_decision8_workspace asks for");
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
    plan_decision8(x->rows, y->rows, D, C, a);
    const hipStream_t s = (hipStream_t)stream;
    const unsigned joins = (unsigned)((x->rows * C + 255) / 256);
    if (y->rows == 0) {
        a.splits = 0;
        hipLaunchKernelGGL(decision8_join_kernel, dim3(joins), dim3(256), 0, s, a);
        QK_HIP(hipGetLastError());
        return QK_OK;
    }
    hipLaunchKernelGGL(decision8_wave_kernel, dim3((unsigned)((x->rows + 31) / 32), (unsigned)a.splits), dim3(256),
                       (size_t)4 * 32 * C * sizeof(float), s, a);
    QK_HIP(hipGetLastError());
    if (a.splits > 1) {
        hipLaunchKernelGGL(decision8_join_kernel, dim3(joins), dim3(256), 0, s, a);
        QK_HIP(hipGetLastError());
    }
    return QK_OK;
}
