// The end of one block and the beginning of the next, row by row of K channels:
//   b = x, or x / sqrt(mean(x^2) + eps) * branch_weight;   h = residual_scale * residual + gate * b  (h = gate * b without a residual)
//   y = (h - m) / sqrt(mean((h - m)^2) + eps) * weight * (1 + scale) + shift,   m = 0 (RMS norm) or mean(h) (layer norm)
// Vectors that are not given are left out.  gate, scale and shift belong to a batch entry, a packed sequence or a token.  All of it is fp32 from
// the first conversion to the last: y is made of h as it is, before h is rounded for the residual stream.
// The mean is taken before the deviations' squares are summed, from registers: their difference in one pass would lose what a large mean leaves.  So would the
// mean's own rounding, 2^-24 of it beside a spread that may be less: the deviations are summed with their squares, and what they have in common is taken out of both.
// Squares whose sum leaves fp32's range, at either end, are summed once more in 64 bits: rows of finite numbers have finite norms.
// Bound by the traffic, 8 bytes an element with a residual: 2 x 4608 x 5120 72 us, 5.2 TB/s (a copy reaches 5.1 here), 4096 x 4096 21.6, 6.2 TB/s; one row of 4096 with
// both norms 2.8, launch and latencies.
#include "svdq_common.h"

using namespace svdq;

namespace {

struct NormParams {
    const char *x, *residual, *weight, *branch_weight, *gate, *scale, *shift;
    char *y, *h;
    const int *cu_seqlens;
    long long first, M, ld_x, ld_residual, ld_y, ld_h;   // bytes; rows first .. M are this launch's
    long long gate_s[2], scale_s[2], shift_s[2];        // bytes: entry, token
    long long tokens;                                   // rows of an entry
    int sequences, pieces, zero_rest;                   // pieces of 8 elements per row
    float inv_k, tiny, eps, residual_scale;
};

template <bool BF16>
__device__ inline void unpack(const u32x4_t w, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t pair = w[j];
        if (BF16) {
            f[2 * j] = bits_f32(pair << 16);
            f[2 * j + 1] = bits_f32(pair & 0xFFFF0000u);
        } else {
            const half2_t h = __builtin_bit_cast(half2_t, pair);
            f[2 * j] = (float)h[0];
            f[2 * j + 1] = (float)h[1];
        }
    }
}
template <bool BF16>
__device__ inline u32x4_t pack(const float (&f)[8]) {
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (BF16) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
        else w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j + 1]) << 16);
    }
    return w;
}

// x of 16 lanes, of 64, added, in all of them
template <int CONTROL>
__device__ inline float moved(float x) {
    return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), CONTROL, 0xF, 0xF, true));
}
__device__ inline float sum16(float x) {
    x += moved<0xB1>(x);  // (quads, then mirrored halves of 8 and of 16)
    x += moved<0x4E>(x);
    x += moved<0x141>(x);
    return x + moved<0x140>(x);
}
__device__ inline float sum64(float x) {
    x = sum16(x);
    const auto a = __builtin_amdgcn_permlane16_swap(f32_bits(x), f32_bits(x), false, false);
    x = bits_f32(a[0]) + bits_f32(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
    return bits_f32(b[0]) + bits_f32(b[1]);
}
__device__ inline double sum16(double x) {
#pragma unroll
    for (int d = 8; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
__device__ inline double sum64(double x) {
    x = sum16(x);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// The sum of x over a row's threads, in all of them.  WIDE: a workgroup has the row; `slot`: a place in LDS of its own for every sum, so that one barrier each is enough
template <bool WIDE, typename T>
__device__ inline T row_sum(T x, T (*place)[16], int slot) {
    x = sum64(x);
    if constexpr (WIDE) {
        const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
        if (lane == 0) place[slot][threadIdx.x >> 6] = x;
        __syncthreads();
        x = sum16((lane & 15) < waves ? place[slot][lane & 15] : (T)0);
    }
    return x;
}

// Those of x and y, in places `slot` and the next.  The half-waves exchange first, so that one has x left and the other y: both cost what one does
// (two sums one beside the other: 2 x 1157 x 2304 7.2 us, this 7.0; 9000 x 5120 33.2, 32.4)
template <bool WIDE>
__device__ inline void row_sums(float &x, float &y, float (*place)[16], int slot) {
    const auto a = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(y), false, false);
    float s = sum16(bits_f32(a[0]) + bits_f32(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(f32_bits(s), f32_bits(s), false, false);
    s = bits_f32(b[0]) + bits_f32(b[1]);
    if constexpr (WIDE) {
        const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
        float *mine = place[slot + (lane >> 5)];
        if ((lane & 31) == 0) mine[threadIdx.x >> 6] = s;
        __syncthreads();
        s = sum16((lane & 15) < waves ? mine[lane & 15] : 0.f);
    }
    x = bits_f32(__builtin_amdgcn_readlane(f32_bits(s), 0));
    y = bits_f32(__builtin_amdgcn_readlane(f32_bits(s), 32));
}

// h <- (h - m) / sqrt(mean((h - m)^2) + eps), the pieces of this thread that lie in the row
template <bool WIDE, int VECS, bool CENTER>
__device__ inline void normalise(float (&h)[VECS][8], const NormParams &p, int t, int threads, int slot) {
    __shared__ float sums[5][16];
    __shared__ double wide[4][16];
    float m = 0.f;
    if constexpr (CENTER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) s += h[i][j];  // (zeros behind the row's end)
        m = row_sum<WIDE>(s, sums, slot) * p.inv_k;
    }
    float squares = 0.f, rest = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        if (t + i * threads >= p.pieces) break;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = h[i][j] - m;
            squares = __builtin_fmaf(d, d, squares);
            if (CENTER) rest += d;
        }
    }
    bool good = true;
    if constexpr (CENTER) {
        row_sums<WIDE>(squares, rest, sums, slot + 1);
        const float common = rest * (rest * p.inv_k);
        good = common <= 0.5f * squares;  // (else next to nothing is left of the squares, as of a row of equal numbers; or a NaN)
        rest *= p.inv_k;
        squares -= common;
    } else {
        squares = row_sum<WIDE>(squares, sums, slot + 1);
    }
    if (good && squares < 0x1p120f && squares >= p.tiny) {
        const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(squares, p.inv_k, p.eps)), c = -rest * r;
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) h[i][j] = CENTER ? __builtin_fmaf(h[i][j] - m, r, c) : h[i][j] * r;
        return;
    }
    const double inv_k = 1.0 / (8.0 * p.pieces);
    double mean = 0.0, s = 0.0;
    if constexpr (CENTER) {
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) s += (double)h[i][j];
        mean = row_sum<WIDE>(s, wide, slot) * inv_k;
        s = 0.0;
    }
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        if (t + i * threads >= p.pieces) break;
#pragma unroll
        for (int j = 0; j < 8; j++) s += ((double)h[i][j] - mean) * ((double)h[i][j] - mean);
    }
    const double r = 1.0 / __builtin_sqrt(row_sum<WIDE>(s, wide, slot + 1) * inv_k + (double)p.eps);
#pragma unroll
    for (int i = 0; i < VECS; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = (float)(((double)h[i][j] - mean) * r);
}

// The sequence of a row: how many offsets are not behind it, less one (-1 or the number of sequences: none), 64 at a time
__device__ inline int sequence_of(const NormParams &p, long long row) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int base = 0; base <= p.sequences; base += 64) n += __popcll(__ballot(base + lane <= p.sequences && p.cu_seqlens[base + lane] <= row));
    return n - 1;
}

// A row to a wave, four to a workgroup, or (WIDE) to a workgroup; each thread up to VECS pieces of 8 elements.  Of rows of one piece a thread, everything is asked for
// at once.
template <bool BF16, bool WIDE, int VECS, bool LAYER>
__global__ void __launch_bounds__(WIDE ? 1024 : 256) gated_norm_kernel(NormParams p) {
    constexpr bool EARLY = VECS == 1;
    const int threads = WIDE ? blockDim.x : 64, t = WIDE ? threadIdx.x : threadIdx.x & 63;
    const long long row = p.first + (WIDE ? blockIdx.x : (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    if (row >= p.M) return;  // (all threads of a row)
    u32x4_t w[VECS], r[VECS];
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int piece = t + i * threads;
        w[i] = r[i] = u32x4_t{0, 0, 0, 0};
        if (piece < p.pieces) {
            w[i] = *(const u32x4_t *)(p.x + row * p.ld_x + (size_t)piece * 16);
            if (p.residual) r[i] = *(const u32x4_t *)(p.residual + row * p.ld_residual + (size_t)piece * 16);
        }
    }
    int entry = 0, token = 0;
    if (p.cu_seqlens) {
        entry = sequence_of(p, row);
        if (entry < 0 || entry >= p.sequences) {
#pragma unroll
            for (int i = 0; i < VECS; i++) {
                const int piece = t + i * threads;
                if (piece >= p.pieces) break;
                if (p.zero_rest & 1) *(u32x4_t *)(p.y + row * p.ld_y + (size_t)piece * 16) = u32x4_t{0, 0, 0, 0};
                if (p.h && (p.zero_rest & 2)) *(u32x4_t *)(p.h + row * p.ld_h + (size_t)piece * 16) = u32x4_t{0, 0, 0, 0};
            }
            return;
        }
    } else if (p.gate || p.scale || p.shift) {
        entry = (int)row / (int)p.tokens;
        token = (int)row - entry * (int)p.tokens;
    }
    const char *vectors[5] = {p.branch_weight, p.gate, p.weight, p.scale, p.shift};
    if (p.gate) vectors[1] += entry * p.gate_s[0] + token * p.gate_s[1];
    if (p.scale) vectors[3] += entry * p.scale_s[0] + token * p.scale_s[1];
    if (p.shift) vectors[4] += entry * p.shift_s[0] + token * p.shift_s[1];
    u32x4_t early[EARLY ? 5 : 1];
    if constexpr (EARLY) {
#pragma unroll
        for (int v = 0; v < 5; v++) {
            early[v] = u32x4_t{0, 0, 0, 0};
            if (vectors[v] && t < p.pieces) early[v] = *(const u32x4_t *)(vectors[v] + (size_t)t * 16);
        }
    }
    float h[VECS][8], f[8];
#pragma unroll
    for (int i = 0; i < VECS; i++) unpack<BF16>(w[i], h[i]);
    // f: of vector v, this thread's piece i
    auto piece_of = [&](int v, int i) __attribute__((always_inline)) {
        if constexpr (EARLY) unpack<BF16>(early[v], f);
        else unpack<BF16>(*(const u32x4_t *)(vectors[v] + (size_t)(t + i * threads) * 16), f);
    };
    auto times = [&](int v, float add) __attribute__((always_inline)) {
        if (!vectors[v]) return;
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            if (t + i * threads >= p.pieces) break;
            piece_of(v, i);
#pragma unroll
            for (int j = 0; j < 8; j++) h[i][j] *= add + f[j];
        }
    };
    if (p.branch_weight) {
        normalise<WIDE, VECS, false>(h, p, t, threads, 0);
        times(0, 0.f);
    }
    times(1, 0.f);
    if (p.residual) {
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const int piece = t + i * threads;
            unpack<BF16>(r[i], f);
#pragma unroll
            for (int j = 0; j < 8; j++) h[i][j] = __builtin_fmaf(p.residual_scale, f[j], h[i][j]);
            if (piece < p.pieces && p.h) *(u32x4_t *)(p.h + row * p.ld_h + (size_t)piece * 16) = pack<BF16>(h[i]);
        }
    }
    normalise<WIDE, VECS, LAYER>(h, p, t, threads, 2);
    times(2, 0.f);
    times(3, 1.f);
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int piece = t + i * threads;
        if (piece >= p.pieces) break;
        if (p.shift) {
            piece_of(4, i);
#pragma unroll
            for (int j = 0; j < 8; j++) h[i][j] += f[j];
        }
        *(u32x4_t *)(p.y + row * p.ld_y + (size_t)piece * 16) = pack<BF16>(h[i]);
    }
}

template <bool BF16, bool WIDE, int VECS>
void launch_rows(const NormParams &p, int threads, bool layer, hipStream_t st) {
    const long long rows = p.M - p.first;
    const dim3 grid((unsigned)(WIDE ? rows : (rows + 3) / 4)), block(WIDE ? threads : 256);
    if (layer) SVDQ_LAUNCH((gated_norm_kernel<BF16, WIDE, VECS, true>), grid, block, 0, st, p);
    else SVDQ_LAUNCH((gated_norm_kernel<BF16, WIDE, VECS, false>), grid, block, 0, st, p);
}

template <bool BF16>
void dispatch(const NormParams &p, bool layer, hipStream_t st) {
    const int need = p.pieces, waves = (need + 63) / 64;
    // Two pieces a thread, where there is no residual to be asked for beside the row, if the rows are more than the card takes at once.  Us, two / one: 9000 x 5120 30.4 / 41.7,
    // 4096 x 4096 13.3 / 14.4, 700 x 4096 4.9 / 5.0; 1500 x 1536 4.8 / 4.5; with a residual 16384 x 1536 32.5 / 30.2, 4096 x 4096 22.6 / 21.6
    const bool two = !p.residual && waves > 2 && (p.M - p.first) * need > 320000;
    if (waves == 1) launch_rows<BF16, false, 1>(p, 64, layer, st);
    else if (waves <= 16 && !two) launch_rows<BF16, true, 1>(p, waves * 64, layer, st);
    else if (waves <= 32) launch_rows<BF16, true, 2>(p, (waves + 1) / 2 * 64, layer, st);
    else launch_rows<BF16, true, 4>(p, (waves + 3) / 4 * 64, layer, st);
}

bool vector_ok(const void *v, const int64_t *s) { return !v || ((uintptr_t)v % 16 == 0 && s[0] >= 0 && s[1] >= 0 && (s[0] | s[1]) % 8 == 0); }

}  // namespace

extern "C" int svdq_gated_norm(const svdq_gated_norm_args *a, void *stream) {
    SVDQ_REQUIRE(a && a->input && a->output, "gated_norm: input and output must not be null");
    SVDQ_REQUIRE(a->residual || !a->residual_out, "gated_norm: residual_out is the sum with a residual, which must not be null");
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "gated_norm: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", (int)a->dtype);
    SVDQ_REQUIRE(a->M > 0 && a->M < (1ll << 31), "gated_norm: M (%lld) must be in 1..2^31-1", (long long)a->M);
    SVDQ_REQUIRE(a->K > 0 && a->K <= 32768 && a->K % 8 == 0, "gated_norm: K (%lld) must be a multiple of 8 up to 32768", (long long)a->K);
    const struct {
        const char *name;
        const void *p;
        int64_t ld;
    } rows[] = {{"input", a->input, a->ld_input}, {"residual", a->residual, a->ld_residual}, {"output", a->output, a->ld_output}, {"residual_out", a->residual_out, a->ld_residual_out}};
    for (const auto &r : rows) {
        if (!r.p) continue;
        SVDQ_REQUIRE((uintptr_t)r.p % 16 == 0, "gated_norm: %s must be 16-byte aligned", r.name);
        SVDQ_REQUIRE(r.ld >= a->K && r.ld % 8 == 0, "gated_norm: rows of %s must be at least K elements and a multiple of 8 apart, got %lld", r.name, (long long)r.ld);
    }
    SVDQ_REQUIRE(((uintptr_t)a->weight | (uintptr_t)a->branch_weight) % 16 == 0, "gated_norm: weight and branch_weight must be 16-byte aligned");
    SVDQ_REQUIRE(vector_ok(a->gate, a->gate_stride) && vector_ok(a->scale, a->scale_stride) && vector_ok(a->shift, a->shift_stride),
                 "gated_norm: gate, scale and shift must be 16-byte aligned, their strides multiples of 8");
    if (a->cu_seqlens) {
        SVDQ_REQUIRE((uintptr_t)a->cu_seqlens % 4 == 0 && a->sequences > 0 && a->sequences < (1ll << 24), "gated_norm: cu_seqlens must be 4-byte aligned, sequences (%lld) in 1..2^24-1",
                     (long long)a->sequences);
    } else {
        SVDQ_REQUIRE(a->tokens > 0, "gated_norm: tokens (%lld), the rows of a batch entry, must be positive", (long long)a->tokens);
    }
    SVDQ_REQUIRE(a->eps >= 0.f && a->eps < __builtin_huge_valf(), "gated_norm: eps must be a finite number not below zero");
    SVDQ_REQUIRE(a->residual_scale - a->residual_scale == 0.f, "gated_norm: residual_scale must be finite");
    NormParams p;
    p.x = (const char *)a->input;
    p.residual = (const char *)a->residual;
    p.weight = (const char *)a->weight;
    p.branch_weight = (const char *)a->branch_weight;
    p.gate = (const char *)a->gate;
    p.scale = (const char *)a->scale;
    p.shift = (const char *)a->shift;
    p.y = (char *)a->output;
    p.h = (char *)a->residual_out;
    p.cu_seqlens = a->cu_seqlens;
    p.ld_x = a->ld_input * 2;
    p.ld_residual = a->ld_residual * 2;
    p.ld_y = a->ld_output * 2;
    p.ld_h = a->ld_residual_out * 2;
    for (int i = 0; i < 2; i++) {
        p.gate_s[i] = a->gate_stride[i] * 2;
        p.scale_s[i] = a->scale_stride[i] * 2;
        p.shift_s[i] = a->shift_stride[i] * 2;
    }
    p.tokens = a->cu_seqlens || a->tokens > a->M ? a->M : a->tokens;  // (32 bits hold it)
    p.sequences = (int)a->sequences;
    p.pieces = (int)(a->K / 8);
    p.zero_rest = a->zero_rest;
    p.inv_k = 1.0f / (float)a->K;
    // fp32 rounds a square by 2^-150 at most, K of them by K * 2^-150: from K * 2^-126 on 2^-24 of the sum, and nothing beside an eps of 2^-120
    p.tiny = a->eps >= 0x1p-120f ? 0.f : 0x1p-100f;
    p.eps = a->eps;
    p.residual_scale = a->residual_scale;
    // a launch takes fewer than 2^32 threads
    const long long most = 1ll << 21;
    for (p.first = 0; p.first < a->M; p.first += most) {
        p.M = a->M - p.first < most ? a->M : p.first + most;
        if (a->dtype == SVDQ_BF16) dispatch<true>(p, a->layer != 0, (hipStream_t)stream);
        else dispatch<false>(p, a->layer != 0, (hipStream_t)stream);
        if (int rc = check_launch("gated_norm")) return rc;
    }
    return SVDQ_OK;
}
