// Rotary positions with several axes, behind the RMS norm of every head where its weights are given: channels come in pairs, (2 i, 2 i + 1) or
// (i, i + R / 2) of the R rotated channels of a head, and the pairs in runs, one for each axis of the positions (time, height, width).  With the
// angle phi = position[axis] * frequency[pair] a pair (x, y) becomes (x cos phi - y sin phi, x sin phi + y cos phi).  Channels behind the R pass.
//
// Angles.  A frequency in revolutions, theta^(-e) / (2 pi), comes from the host in two parts, 64 bits and the next ones: one of 53 bits alone would leave 2^-22
// radians of a position of 2^31 open, more than fp32 rounds by.  The product's high part loses its whole revolutions before the low ones are added.  What is
// left open is what 80 bits leave of the frequency on the host, 2^-55 of the angle at most (2^-24 radians at 2^31).  Sine and cosine see half a revolution at most.
// They are the same for all heads of a token: a wave makes those of its token once, a pair to a lane, and hands them round through LDS.
#include <math.h>

#include "svdq_common.h"

using namespace svdq;

namespace {

constexpr int MAX_PAIRS = 128, MAX_AXES = 4, ITEMS = 4;

struct RotaryParams {
    const char *in[2], *norm[2];   // q, k
    char *out[2];
    const void *positions;
    long long in_s[2][3], out_s[2][3];  // bytes: batch, token, head
    long long pos_s[3];                 // elements: batch, token, axis
    long long work, first;              // tokens of all entries times the waves that share one; this launch's first
    int T, heads[2], D, pairs, halves, position_type, share;  // share: waves to a token
    int once;                           // the tensors do not fit the memory-side cache: what is read is not kept there
    float inv_d, eps, tiny;
    double freq[MAX_PAIRS];  // revolutions per position
    float low[MAX_PAIRS];    // what 64 bits leave of them
    uint8_t axis[MAX_PAIRS];
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

// x of the lanes that share a head, added: within quads, then mirrored halves of 8 and of 16
template <int CONTROL>
__device__ inline float moved(float x) {
    return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), CONTROL, 0xF, 0xF, true));
}
template <int LANES>
__device__ inline float head_sum(float x) {
    x += moved<0xB1>(x);
    x += moved<0x4E>(x);
    if (LANES > 4) x += moved<0x141>(x);
    if (LANES > 8) x += moved<0x140>(x);
    if (LANES > 16) x += __shfl_xor(x, 16);
    return x;
}

// A wave to a token, or several, each with some of its heads: 64 / LANES heads at a time, LANES threads to a head, a piece of 8 channels each, ITEMS times on their way.
template <bool BF16, int LANES, bool NORM, bool HALVES>
__global__ void __launch_bounds__(256) rotary_axes_kernel(RotaryParams p) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    __shared__ __attribute__((aligned(16))) float2_t table[4][MAX_PAIRS];  // cosine, sine
    constexpr int SLOTS = 64 / LANES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LANES, slot = lane / LANES;
    const long long at = p.first + (long long)blockIdx.x * 4 + wave;
    if (at >= p.work) return;
    const int row = (int)(at / p.share), part = (int)(at - (long long)row * p.share), b = row / p.T, t = row - b * p.T;
    const bool in = c < p.D / 8;
    // turns of SLOTS heads: those of q, then those of k
    const int nq = (p.heads[0] + SLOTS - 1) / SLOTS, all = nq + (p.heads[1] + SLOTS - 1) / SLOTS;
    int turn = part * all / p.share;
    const int end = (part + 1) * all / p.share;
    // This lane's piece of a turn's head, in and out, moved on turn by turn: from q's last one to k's first
    const char *first_in[2];
    char *first_out[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        first_in[k] = p.in[k] + b * p.in_s[k][0] + t * p.in_s[k][1] + (slot * p.in_s[k][2] + c * 16);
        first_out[k] = p.out[k] + b * p.out_s[k][0] + t * p.out_s[k][1] + (slot * p.out_s[k][2] + c * 16);
    }
    const int begun = turn < nq ? turn : turn - nq;
    const char *src = (turn < nq ? first_in[0] : first_in[1]) + begun * SLOTS * (turn < nq ? p.in_s[0][2] : p.in_s[1][2]);
    char *dst = (turn < nq ? first_out[0] : first_out[1]) + begun * SLOTS * (turn < nq ? p.out_s[0][2] : p.out_s[1][2]);
    // whether this lane has a piece of turn x
    auto has = [&](int x) __attribute__((always_inline)) {
        const int left = x < nq ? p.heads[0] - x * SLOTS : p.heads[1] - (x - nq) * SLOTS;
        return in && slot < left;
    };
    u32x4_t w[ITEMS];
    auto load = [&](int first) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            w[i] = u32x4_t{0, 0, 0, 0};
            if (first + i >= end) continue;
            if (has(first + i)) {
                if (p.once) w[i] = __builtin_nontemporal_load((const u32x4_t *)src);
                else w[i] = *(const u32x4_t *)src;
            }
            src += SLOTS * (first + i < nq ? p.in_s[0][2] : p.in_s[1][2]);
            if (first + i == nq - 1) src = first_in[1];
        }
    };
    load(turn);
    u32x4_t g[2];
    if (NORM) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            g[k] = u32x4_t{0, 0, 0, 0};
            if (p.norm[k] && in) g[k] = *(const u32x4_t *)(p.norm[k] + c * 16);
        }
    }
    for (int pair = lane; pair < p.pairs; pair += 64) {
        const long long from = b * p.pos_s[0] + t * p.pos_s[1] + p.axis[pair] * p.pos_s[2];
        const double freq = p.freq[pair], low = (double)p.low[pair];
        auto fraction = [&](double x) __attribute__((always_inline)) {  // of x positions' revolutions
            const double whole = x * freq, r = (whole - __builtin_rint(whole)) + (__builtin_fma(x, freq, -whole) + x * low);
            return r - __builtin_rint(r);
        };
        double r;
        if (p.position_type == SVDQ_POSITION_INT64) {
            const int64_t x = ((const int64_t *)p.positions)[from], rest = x < 1ll << 53 && x > -(1ll << 53) ? 0 : x & 2047;  // (the rest fits 64 bits)
            r = fraction((double)(x - rest));
            if (rest) {
                r += fraction((double)rest);
                r -= __builtin_rint(r);
            }
        } else {
            r = fraction(p.position_type == SVDQ_POSITION_INT32 ? (double)((const int32_t *)p.positions)[from] : (double)((const float *)p.positions)[from]);
        }
        float s, co;
        sincospif(2.0f * (float)r, &s, &co);
        table[wave][pair] = float2_t{co, s};
    }
    __builtin_amdgcn_wave_barrier();  // (LDS serves a wave in order)
    // this lane's channels: of pair j cosine and sine; (1, 0) where channels pass
    constexpr int PAIRS = HALVES ? 8 : 4;
    const int half = p.pairs / 8;
    const bool low = c < half;
    float co[PAIRS], si[PAIRS];
#pragma unroll
    for (int j = 0; j < PAIRS; j++) {
        const int pair = HALVES ? (low ? c : c - half) * 8 + j : c * 4 + j;
        const bool turned = HALVES ? c < 2 * half : pair < p.pairs;
        const float2_t cs = table[wave][turned ? pair : 0];
        co[j] = turned ? cs[0] : 1.f;
        si[j] = turned ? cs[1] : 0.f;
        if (HALVES && low) si[j] = -si[j];
    }
    for (; turn < end; turn += ITEMS) {
        if (turn != part * all / p.share) load(turn);
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            if (turn + i >= end) break;
            const int k = turn + i >= nq;
            float x[8], y[8];
            unpack<BF16>(w[i], x);
            if (NORM && p.norm[k]) {
                float squares = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) squares = __builtin_fmaf(x[j], x[j], squares);
                squares = head_sum<LANES>(squares);
                if (squares < 0x1p120f && squares >= p.tiny) {
                    const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(squares, p.inv_d, p.eps));
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] *= r;
                } else {  // squares that leave fp32's range: once more in 64 bits (all lanes of the head)
                    double s = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; j++) s += (double)x[j] * (double)x[j];
#pragma unroll
                    for (int d = LANES / 2; d; d >>= 1) s += __shfl_xor(s, d);
                    const double r = 1.0 / __builtin_sqrt(s / (double)p.D + (double)p.eps);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = (float)((double)x[j] * r);
                }
                unpack<BF16>(g[k], y);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] *= y[j];
            }
            if (HALVES) {
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = __shfl(x[j], low ? c + half : c - half, LANES);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = c < 2 * half ? x[j] * co[j] + y[j] * si[j] : x[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float a = x[2 * j], d = x[2 * j + 1];
                    x[2 * j] = a * co[j] - d * si[j];
                    x[2 * j + 1] = a * si[j] + d * co[j];
                }
            }
            if (has(turn + i)) *(u32x4_t *)dst = pack<BF16>(x);
            dst += SLOTS * (k ? p.out_s[1][2] : p.out_s[0][2]);
            if (turn + i == nq - 1) dst = first_out[1];
        }
    }
}

template <bool BF16, int LANES, bool NORM>
void launch_pairs(const RotaryParams &p, unsigned blocks, hipStream_t st) {
    if (p.halves) SVDQ_LAUNCH((rotary_axes_kernel<BF16, LANES, NORM, true>), dim3(blocks), dim3(256), 0, st, p);
    else SVDQ_LAUNCH((rotary_axes_kernel<BF16, LANES, NORM, false>), dim3(blocks), dim3(256), 0, st, p);
}
template <bool BF16, int LANES>
void launch_lanes(const RotaryParams &p, unsigned blocks, hipStream_t st) {
    if (p.norm[0] || p.norm[1]) launch_pairs<BF16, LANES, true>(p, blocks, st);
    else launch_pairs<BF16, LANES, false>(p, blocks, st);
}
template <bool BF16>
void dispatch(const RotaryParams &p, unsigned blocks, hipStream_t st) {
    if (p.D <= 32) launch_lanes<BF16, 4>(p, blocks, st);
    else if (p.D <= 64) launch_lanes<BF16, 8>(p, blocks, st);
    else if (p.D <= 128) launch_lanes<BF16, 16>(p, blocks, st);
    else launch_lanes<BF16, 32>(p, blocks, st);
}

}  // namespace

extern "C" int svdq_rotary_axes(const svdq_rotary_axes_args *a, void *stream) {
    SVDQ_REQUIRE(a && a->q && a->q_out && a->positions, "rotary_axes: q, q_out and positions must not be null");
    SVDQ_REQUIRE(!a->k == !a->k_out && (a->k || !a->norm_k), "rotary_axes: k, k_out and norm_k belong together");
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "rotary_axes: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", (int)a->dtype);
    SVDQ_REQUIRE(a->position_type >= SVDQ_POSITION_INT32 && a->position_type <= SVDQ_POSITION_FP32, "rotary_axes: position_type %d is unknown", (int)a->position_type);
    SVDQ_REQUIRE(a->batch > 0 && a->tokens > 0 && a->batch < (1ll << 31) && a->tokens < (1ll << 31) && a->batch * a->tokens < (1ll << 31),
                 "rotary_axes: batch (%lld) times tokens (%lld) must be in 1..2^31-1", (long long)a->batch, (long long)a->tokens);
    SVDQ_REQUIRE(a->heads > 0 && a->heads < 65536 && (!a->k || (a->kv_heads > 0 && a->kv_heads < 65536)), "rotary_axes: heads (%lld, %lld) must be in 1..65535", (long long)a->heads,
                 (long long)a->kv_heads);
    SVDQ_REQUIRE(a->head_dim > 0 && a->head_dim <= 2 * MAX_PAIRS && a->head_dim % 8 == 0, "rotary_axes: head_dim (%lld) must be a multiple of 8 up to 256", (long long)a->head_dim);
    SVDQ_REQUIRE(a->axes > 0 && a->axes <= MAX_AXES, "rotary_axes: axes (%lld) must be in 1..4", (long long)a->axes);
    int64_t rotated = 0;
    for (int i = 0; i < a->axes; i++) {
        SVDQ_REQUIRE(a->axis_dim[i] > 0 && a->axis_dim[i] % 2 == 0 && a->axis_dim[i] <= a->head_dim, "rotary_axes: axis_dim[%d] (%lld) must be even and positive", i, (long long)a->axis_dim[i]);
        SVDQ_REQUIRE(a->theta[i] > 0.0 && a->theta[i] < __builtin_huge_val(), "rotary_axes: theta must be a positive number");
        rotated += a->axis_dim[i];
    }
    SVDQ_REQUIRE(rotated <= a->head_dim, "rotary_axes: the axes' channels (%lld) must not be more than head_dim (%lld)", (long long)rotated, (long long)a->head_dim);
    SVDQ_REQUIRE(!a->halves || rotated % 16 == 0, "rotary_axes: halves of the rotated channels (%lld) must be multiples of 8", (long long)rotated);
    for (int i = 0; i < 3; i++)
        SVDQ_REQUIRE(a->q_stride[i] >= 0 && a->k_stride[i] >= 0 && a->q_out_stride[i] >= 0 && a->k_out_stride[i] >= 0 &&
                         (a->q_stride[i] | a->k_stride[i] | a->q_out_stride[i] | a->k_out_stride[i]) % 8 == 0,
                     "rotary_axes: strides must be multiples of 8 elements (16 bytes)");
    SVDQ_REQUIRE(a->position_stride[0] >= 0 && a->position_stride[1] >= 0 && a->position_stride[2] >= 0, "rotary_axes: strides of positions must not be negative");
    SVDQ_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->q_out | (uintptr_t)a->k_out | (uintptr_t)a->norm_q | (uintptr_t)a->norm_k) % 16 == 0,
                 "rotary_axes: pointers must be 16-byte aligned");
    SVDQ_REQUIRE((uintptr_t)a->positions % (a->position_type == SVDQ_POSITION_INT64 ? 8 : 4) == 0, "rotary_axes: positions must be aligned to their type");
    SVDQ_REQUIRE(a->eps >= 0.f && a->eps < __builtin_huge_valf(), "rotary_axes: eps must be a finite number not below zero");
    RotaryParams p;
    const void *ins[2] = {a->q, a->k}, *norms[2] = {a->norm_q, a->norm_k};
    void *outs[2] = {a->q_out, a->k_out};
    const int64_t *in_s[2] = {a->q_stride, a->k_stride}, *out_s[2] = {a->q_out_stride, a->k_out_stride};
    for (int i = 0; i < 2; i++) {
        p.in[i] = (const char *)ins[i];
        p.norm[i] = (const char *)norms[i];
        p.out[i] = (char *)outs[i];
        for (int j = 0; j < 3; j++) {
            p.in_s[i][j] = in_s[i][j] * 2;
            p.out_s[i][j] = out_s[i][j] * 2;
        }
    }
    p.positions = a->positions;
    for (int j = 0; j < 3; j++) p.pos_s[j] = a->position_stride[j];
    p.T = (int)a->tokens;
    p.heads[0] = (int)a->heads;
    p.heads[1] = a->k ? (int)a->kv_heads : 0;
    p.D = (int)a->head_dim;
    p.pairs = (int)(rotated / 2);
    p.halves = a->halves != 0;
    p.position_type = a->position_type;
    p.inv_d = 1.0f / (float)a->head_dim;
    p.eps = a->eps;
    p.tiny = a->eps >= 0x1p-120f ? 0.f : 0x1p-100f;
    // An axis' frequencies are a geometric series.  80 bits round by 2^-64: number j is off by 3 j of that for the products and the step's exponential, by 3 e log(theta) for the
    // logarithm and the exponent, and by 4, which for 128 pairs and any theta up to 10^15 is less than 2^-55
    int pair = 0;
    for (int i = 0; i < a->axes; i++) {
        const long double span = a->whole_spectrum ? (long double)rotated : (long double)a->axis_dim[i], rate = -logl((long double)a->theta[i]);
        const long double step = expl(rate * 2.0L / span);
        long double f = (a->whole_spectrum ? expl(rate * 2.0L * pair / span) : 1.0L) / 6.283185307179586476925286766559L;
        for (int j = 0; j < a->axis_dim[i] / 2; j++, pair++, f *= step) {
            p.freq[pair] = (double)f;
            p.low[pair] = f < 0x1p170L ? (float)(f - (long double)p.freq[pair]) : 0.f;  // (those beyond, of a theta near zero, have nothing left of their angles)
            p.axis[pair] = (uint8_t)i;
        }
    }
    const int lanes = p.D <= 32 ? 4 : p.D <= 64 ? 8 : p.D <= 128 ? 16 : 32, slots = 64 / lanes, turns = (p.heads[0] + slots - 1) / slots + (p.heads[1] + slots - 1) / slots;
    const long long rows = a->batch * a->tokens;
    // Four waves to a SIMD, as far as there is a turn for each: fewer leave latencies bare (8 tokens, 40 heads of 128 a wave to a token 7.7 us, to a turn 4.4), more are more of
    // what every wave does for its angles (2 x 1157, 32 heads of 80 with eight 12.3, with four 10.1, with two 11.1)
    p.share = 1;
    while (rows * p.share < 4096 && p.share < turns) p.share++;
    p.work = rows * p.share;
    p.once = rows * (p.heads[0] + p.heads[1]) * p.D * 4 > 300000000;
    // a launch takes fewer than 2^32 threads, a wave is 64
    const long long most = 1ll << 25, all = p.work;
    for (p.first = 0; p.first < all; p.first += most) {
        p.work = all - p.first < most ? all : p.first + most;
        const unsigned blocks = (unsigned)((p.work - p.first + 3) / 4);
        if (a->dtype == SVDQ_BF16) dispatch<true>(p, blocks, (hipStream_t)stream);
        else dispatch<false>(p, blocks, (hipStream_t)stream);
        if (int rc = check_launch("rotary_axes")) return rc;
    }
    return SVDQ_OK;
}
