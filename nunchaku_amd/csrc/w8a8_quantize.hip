// Rows of bf16 / fp16 activations to 8-bit codes with one scale each, plain or behind a residual's addition and an RMS norm:
//   plain: g = x;   norm: h = T(x + residual) (the stored residual stream; h = x without one), g = h * weight
//   a = max(max_k |g|, 2^-100), code = rne(g * fl32(127 / a)), scale = fl32(a * f / 127), f = 1 or 1 / sqrt(mean(h^2) + eps).
// The factor 1 / rms of a row is the same for all its elements, so it cancels in the codes: they depend on max |g| alone, and
// g is exact in fp32 (two significands of at most 11 bits).  The sum of squares is held in fp32, of h * 2^100 where squares would end below fp32's
// smallest numbers and eps does not make up for them.  |code| <= 127 needs no clamp: |g| * fl32(127 / a) <= 127 (1 + 2^-23).  A row with an
// infinity or a NaN in g (or a sum of squares that is not finite) gets the scale NaN and codes 0: what a product makes of it is NaN.
// Bound by the traffic, 3 bytes per element (7 with a residual): one pass, the row stays in registers.  16384 x 8192 plain 62 us, 6.5 TB/s;
// 9216 x 5120 with residual 53 us, 6.2 TB/s; one row of 4096 2.4 and 2.8 us, launch and latencies.
#include "svdq_common.h"

using namespace svdq;

namespace {

constexpr float MIN_AMAX = 0x1p-100f;
constexpr float TINY_SQUARES = 0x1p-100f;  // fp32 rounds a square by 2^-150 at most, 65536 of them by 2^-134: from here on 2^-34 of the sum

struct QuantizeParams {
    const char *x, *residual, *weight;
    char *residual_out, *codes;
    float *scales;
    long long M, ld_x, ld_residual, ld_residual_out, ld_codes;  // bytes
    int pieces;                                                 // of 8 elements per row
    float inv_k, eps;
    int once;  // the tensors do not fit the memory-side cache: what is read is not kept there
};

// This thread's pieces of a row; zeros behind its end
template <int THREADS, int VECS>
__device__ inline void load_row(u32x4_t (&w)[VECS], const char *row, const QuantizeParams &p, int t) {
#pragma unroll
    for (int i = 0; i < VECS; i++) w[i] = u32x4_t{0, 0, 0, 0};
    if (p.once) {
#pragma unroll
        for (int i = 0; i < VECS; i++)
            if (t + i * THREADS < p.pieces) w[i] = __builtin_nontemporal_load((const u32x4_t *)(row + (size_t)(t + i * THREADS) * 16));
    } else {
#pragma unroll
        for (int i = 0; i < VECS; i++)
            if (t + i * THREADS < p.pieces) w[i] = *(const u32x4_t *)(row + (size_t)(t + i * THREADS) * 16);
    }
}

template <bool BF16>
__device__ inline void unpack(const u32x4_t w, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (BF16) {
            f[2 * j] = bits_f32(w[j] << 16);
            f[2 * j + 1] = bits_f32(w[j] & 0xFFFF0000u);
        } else {
            const uint32_t pair = w[j];  // (a bit cast of w[j] itself takes element 0 whatever j)
            const half2_t h = __builtin_bit_cast(half2_t, pair);
            f[2 * j] = (float)h[0];
            f[2 * j + 1] = (float)h[1];
        }
    }
}
template <bool BF16>
__device__ inline uint32_t pack_pair(float lo, float hi) {
    if (BF16) return pack_bf16x2(lo, hi);
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}

// THREADS per row (32 and 64: several rows per workgroup), each with up to VECS pieces of 8 elements.  A norm without a residual of 1024 threads with four
// pieces fits two workgroups to a compute unit with 64 registers, which the compiler has to be told (2048 x 20000 31.3 -> 23.5 us).
template <bool BF16, int THREADS, int VECS, bool NORM, bool RESIDUAL>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS, THREADS == 1024 && VECS == 4 && NORM && !RESIDUAL ? 8 : THREADS < 256 ? 1 : THREADS / 256)
    quantize_rows_kernel(QuantizeParams p) {
    constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1, WAVES = THREADS <= 64 ? 1 : THREADS / 64;
    const int t = threadIdx.x % THREADS;
    const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / THREADS;
    if (row >= p.M) return;  // (all threads of a row; rows of several waves are one per workgroup)
    u32x4_t w[VECS], r[RESIDUAL ? VECS : 1];
    load_row<THREADS, VECS>(w, p.x + row * p.ld_x, p, t);
    if constexpr (RESIDUAL) load_row<THREADS, VECS>(r, p.residual + row * p.ld_residual, p, t);
    uint32_t top = 0;
    float squares = 0.f;
    u32x4_t nw[NORM ? VECS : 1];
    if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const int piece = t + i * THREADS;
            nw[i] = u32x4_t{0, 0, 0, 0};
            if (piece < p.pieces) nw[i] = *(const u32x4_t *)(p.weight + (size_t)piece * 16);
        }
    }
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int piece = t + i * THREADS;
        float f[8];
        if constexpr (RESIDUAL) {
            float a[8], b[8];
            unpack<BF16>(w[i], a);
            unpack<BF16>(r[i], b);
#pragma unroll
            for (int j = 0; j < 4; j++) w[i][j] = pack_pair<BF16>(a[2 * j] + b[2 * j], a[2 * j + 1] + b[2 * j + 1]);
            if (piece < p.pieces) *(u32x4_t *)(p.residual_out + row * p.ld_residual_out + (size_t)piece * 16) = w[i];
        }
        unpack<BF16>(w[i], f);
        if constexpr (NORM) {
            float g[8];
            unpack<BF16>(nw[i], g);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                squares = __builtin_fmaf(f[j], f[j], squares);
                f[j] *= g[j];
            }
        }
        // magnitudes as integers: NaN is the largest, so that it is not lost
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t m = f32_bits(f[j]) & 0x7FFFFFFFu;
            top = m > top ? m : top;
        }
    }
#pragma unroll
    for (int d = THREADS < 64 ? THREADS / 2 : 32; d; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d);
        top = o > top ? o : top;
        if (NORM) squares += __shfl_xor(squares, d);
    }
    if constexpr (WAVES > 1) {
        __shared__ uint32_t tops[WAVES];
        __shared__ float sums[WAVES];
        if ((t & 63) == 0) {
            tops[t >> 6] = top;
            sums[t >> 6] = squares;
        }
        __syncthreads();
        top = 0;
        squares = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; i++) {
            top = tops[i] > top ? tops[i] : top;
            squares += sums[i];
        }
    }
    const bool bad = top >= 0x7F800000u || !(squares < __builtin_huge_valf());
    const float amax = bits_f32(top) > MIN_AMAX ? bits_f32(top) : MIN_AMAX;
    const float factor = 127.0f / amax;
    if (t == 0) {
        float s = amax;
        if (NORM) s *= 1.0f / __builtin_sqrtf(squares * p.inv_k + p.eps);
        p.scales[row] = bad ? __builtin_nanf("") : s / 127.0f;
    }
    char *out = p.codes + row * p.ld_codes;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int piece = t + i * THREADS;
        float f[8];
        unpack<BF16>(w[i], f);
        if constexpr (NORM) {
            float g[8];
            unpack<BF16>(nw[i], g);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] *= g[j];
        }
        // adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves its two's complement in the low bits
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; j++) b[j] = f32_bits(f[j] * factor + 12582912.0f) & 255u;
        u32x2_t c;
#pragma unroll
        for (int j = 0; j < 2; j++) c[j] = bad ? 0u : b[4 * j] | b[4 * j + 1] << 8 | b[4 * j + 2] << 16 | b[4 * j + 3] << 24;
        if (piece < p.pieces) *(u32x2_t *)(out + (size_t)piece * 8) = c;
    }
    if constexpr (NORM && BF16) {  // (the smallest square in fp16 is 2^-48)
        if (!(p.eps < TINY_SQUARES && squares < TINY_SQUARES)) return;  // (the same in all threads of a row)
        // The squares once more, in units of 2^-200: from 2^-66 on (|h| < 2^-50, in units of 2^-100), sums up to 2^100.  h is read again, this thread's own
        // pieces, and behind the codes: with the row in registers for it the longest ones spilled.
        const char *h = RESIDUAL ? p.residual_out + row * p.ld_residual_out : p.x + row * p.ld_x;
        squares = 0.f;
#pragma unroll 1
        for (int piece = t; piece < p.pieces; piece += THREADS) {
            float f[8];
            unpack<BF16>(*(const u32x4_t *)(h + (size_t)piece * 16), f);
#pragma unroll
            for (int j = 0; j < 8; j++) squares = __builtin_fmaf(f[j] * 0x1p100f, f[j] * 0x1p100f, squares);
        }
#pragma unroll
        for (int d = THREADS < 64 ? THREADS / 2 : 32; d; d >>= 1) squares += __shfl_xor(squares, d);
        if constexpr (WAVES > 1) {
            __shared__ float sums[WAVES];
            if ((t & 63) == 0) sums[t >> 6] = squares;
            __syncthreads();
            squares = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; i++) squares += sums[i];
        }
        // amax is below 2^78 with the largest weight, the root of the mean between 2^-41 and 2^50 (or zero): neither factor leaves fp32
        if (t == 0 && !bad) p.scales[row] = (amax * 0x1p40f) * (0x1p60f / __builtin_sqrtf(squares * p.inv_k + p.eps * 0x1p100f * 0x1p100f)) / 127.0f;
    }
}

template <bool BF16, int THREADS, int VECS>
void launch_rows(const QuantizeParams &p, bool norm, hipStream_t st) {
    constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
    const dim3 grid((unsigned)((p.M + ROWS - 1) / ROWS)), block(THREADS < 256 ? 256 : THREADS);
    if (!norm) SVDQ_LAUNCH((quantize_rows_kernel<BF16, THREADS, VECS, false, false>), grid, block, 0, st, p);
    else if (!p.residual) SVDQ_LAUNCH((quantize_rows_kernel<BF16, THREADS, VECS, true, false>), grid, block, 0, st, p);
    else SVDQ_LAUNCH((quantize_rows_kernel<BF16, THREADS, VECS, true, true>), grid, block, 0, st, p);
}

// The fewest threads that hold a row in one or two pieces each: more of them are more exchanges between waves, more pieces are more work for every
// lane of a row that does not fill them (the last of several pieces of a norm's row is as much work as the first).  Us, this way / the next best,
// 1.3e8 elements, plain and norm with residual: K = 512 73 / 78 (two pieces of 64), 156 / 157; 1024 69 / 70 (four), 159 / 169 (256 threads); 2048 70 / 77
// (four pieces of 64 against 256 threads; with 300 rows 2.9 / 2.7), norm 154 / 168 (256 against four of 64); 4096 69 / 69 (256 threads with four), 154 / 155 (512); 8192 68 / 69, 154 / 155 (512 with four, which
// with 300 rows takes 3.6 and 6.7 against 3.3 and 5.4); 16384 69 / 72, 161 / 158 (512 with four: 300 rows 5.6 and 8.9 against 5.9 and 8.4); 32768 71 / 91, 167 / 191
// (eight pieces).
template <bool BF16>
void dispatch(const QuantizeParams &p, bool norm, hipStream_t st) {
    const int need = p.pieces;
    if (need <= 32) launch_rows<BF16, 32, 1>(p, norm, st);
    else if (need <= 64) launch_rows<BF16, 64, 1>(p, norm, st);
    else if (need <= 64 * 2) launch_rows<BF16, 64, 2>(p, norm, st);
    else if (need <= 64 * 4 && !norm && p.M > 2048) launch_rows<BF16, 64, 4>(p, norm, st);
    else if (need <= 256) launch_rows<BF16, 256, 1>(p, norm, st);
    else if (need <= 256 * 2) launch_rows<BF16, 256, 2>(p, norm, st);
    else if (need <= 512 * 2) launch_rows<BF16, 512, 2>(p, norm, st);
    else if (need <= 1024 * 2) launch_rows<BF16, 1024, 2>(p, norm, st);
    else if (need <= 1024 * 4) launch_rows<BF16, 1024, 4>(p, norm, st);
    else launch_rows<BF16, 1024, 8>(p, norm, st);
}

int quantize_rows(const svdq_quantize_w8a8_args *a, bool norm, void *stream, const char *what) {
    SVDQ_REQUIRE(a && a->input && a->output && a->oscales, "%s: input, output and oscales must not be null", what);
    SVDQ_REQUIRE(!norm || a->weight, "%s: weight must not be null", what);
    SVDQ_REQUIRE(!a->residual == !a->residual_out, "%s: residual and residual_out belong together", what);
    SVDQ_REQUIRE(norm || !a->residual, "%s: takes no residual", what);
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "%s: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", what, (int)a->dtype);
    SVDQ_REQUIRE(a->M > 0 && a->M < (1ll << 31), "%s: M (%lld) must be in 1..2^31-1", what, (long long)a->M);
    SVDQ_REQUIRE(a->K > 0 && a->K <= 65536 && a->K % 16 == 0, "%s: K (%lld) must be a multiple of 16 up to 65536", what, (long long)a->K);
    SVDQ_REQUIRE(a->ld_input >= a->K && a->ld_input % 8 == 0, "%s: rows of input must be at least K elements and a multiple of 8 apart, got %lld", what, (long long)a->ld_input);
    SVDQ_REQUIRE(!a->residual || (a->ld_residual >= a->K && a->ld_residual % 8 == 0), "%s: rows of residual must be at least K elements and a multiple of 8 apart, got %lld", what,
                 (long long)a->ld_residual);
    SVDQ_REQUIRE(!a->residual || (a->ld_residual_out >= a->K && a->ld_residual_out % 8 == 0),
                 "%s: rows of residual_out must be at least K elements and a multiple of 8 apart, got %lld", what, (long long)a->ld_residual_out);
    SVDQ_REQUIRE(((uintptr_t)a->input | (uintptr_t)a->output | (uintptr_t)a->residual | (uintptr_t)a->residual_out | (uintptr_t)a->weight) % 16 == 0,
                 "%s: pointers must be 16-byte aligned", what);
    SVDQ_REQUIRE((uintptr_t)a->oscales % 4 == 0, "%s: oscales must be 4-byte aligned", what);
    SVDQ_REQUIRE(!norm || (a->eps >= 0.f && a->eps < __builtin_huge_valf()), "%s: eps must be a finite number not below zero", what);
    QuantizeParams p;
    p.x = (const char *)a->input;
    p.residual = (const char *)a->residual;
    p.weight = (const char *)a->weight;
    p.residual_out = (char *)a->residual_out;
    p.codes = (char *)a->output;
    p.scales = a->oscales;
    p.M = a->M;
    p.ld_x = a->ld_input * 2;
    p.ld_residual = a->ld_residual * 2;
    p.ld_residual_out = a->ld_residual_out * 2;
    p.ld_codes = a->K;
    p.pieces = (int)(a->K / 8);
    p.inv_k = 1.0f / (float)a->K;
    p.eps = a->eps;
    // Read past the memory-side cache (256 MB) what would not stay there anyway: 16384 x 8192 71 -> 62 us, 9216 x 5120 with residual 57.5 -> 54; where the
    // tensors fit, or nearly, those that another kernel has left there would be fetched again: 16384 x 5600 (275 MB) 45.9 -> 47.3, 9216 x 4096 18.9 -> 20.9,
    // 4608 x 4096 with residual 21.4 -> 24.0
    p.once = a->M * a->K * (a->residual ? 7 : 3) > 300000000;
    // a launch takes fewer than 2^32 threads: 2^31 for so many rows of at most 64 threads, of at most 1024
    const long long most = p.pieces <= 128 ? 1ll << 25 : 1ll << 21;
    for (long long first = 0; first < a->M; first += most) {
        p.M = a->M - first < most ? a->M - first : most;
        if (a->dtype == SVDQ_BF16) dispatch<true>(p, norm, (hipStream_t)stream);
        else dispatch<false>(p, norm, (hipStream_t)stream);
        if (int rc = check_launch(what)) return rc;
        p.x += most * p.ld_x;
        p.codes += most * p.ld_codes;
        p.scales += most;
        if (p.residual) {
            p.residual += most * p.ld_residual;
            p.residual_out += most * p.ld_residual_out;
        }
    }
    return SVDQ_OK;
}

}  // namespace

extern "C" int svdq_quantize_w8a8_act(const svdq_quantize_w8a8_args *args, void *stream) { return quantize_rows(args, false, stream, "quantize_w8a8_act"); }

extern "C" int svdq_rms_norm_quantize_w8a8(const svdq_quantize_w8a8_args *args, void *stream) {
    return quantize_rows(args, true, stream, "rms_norm_quantize_w8a8");
}
