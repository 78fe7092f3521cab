// What the attention kernels share: the matrix instructions of both types, rows of K and V in LDS, the running softmax of 32 rows.
//
// One pass over the keys with the running maximum and sum of the softmax in fp32.  The scores are formed as K q^T on
// v_mfma_f32_32x32x16: a lane then holds 32 keys' scores of ONE row (the other 32 are 32 lanes away), so the maximum and the sum
// take one exchange between lanes, and the scores, rounded to the inputs' type, are the right operand of v^T p^T as they are: the
// instruction contracts 8 keys per lane, which 8 is free, as long as the left operand holds the same.  That operand is v down the
// columns, which LDS reads that transpose 4 x 16 blocks (ds_read_b64_tr_b16) make of plain rows.
//
// Rows of K and V in LDS: pieces of 16 bytes, piece c of row r at place c ^ f(r), so that neither 16 lanes that read one piece of 16
// rows (K) nor 32 lanes that read 64 bytes of 4 rows (V) meet in a bank.
#pragma once

#include "svdq_common.h"

namespace svdq {
namespace attention {

constexpr int KEYS = 64;  // per step

template <bool BF16>
struct Elem;
template <>
struct Elem<true> {
    typedef bf16x8_t vec;
    static constexpr uint32_t ONE = 0x3F80;
    static __device__ inline float16_t mfma(vec a, vec b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ inline uint32_t pair(float lo, float hi) { return pack_bf16x2(lo, hi); }
    static constexpr float RAISED = 0.f;  // as wide a range as fp32
};
template <>
struct Elem<false> {
    typedef half8_t vec;
    static constexpr uint32_t ONE = 0x3C00;
    // Probabilities stand 2^7 times higher than the maximum in use has them, which with the 2^8 that it may lag behind is 2^15 at most.  What a small one
    // loses at the type's end, 2^-25, is then 2^-32 of the sum: one key e^17.5 times as likely as each of 65535 others leaves these 1.6e-3 of the result,
    // all of which was lost without.
    static constexpr float RAISED = 7.f;
    static __device__ inline float16_t mfma(vec a, vec b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ inline uint32_t pair(float lo, float hi) {
        typedef float float2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, half2_t));
    }
};

// A head of DP elements (rounded up): KS steps of 16 in the first product, DB blocks of 32 in the second; rows PITCH bytes apart in LDS.
// Heads of 72 .. 96 take three quarters of the widest rows' LDS (WHOLE: the pitch is a power of two for them, too), which is a third
// workgroup on a compute unit (4096 queries, 256 keys, 4 x 16 heads of 80: 35.9 -> 32.5 us).
template <int DP_, bool WHOLE = false, bool ONES_ = false>
struct Head {
    static constexpr int DP = DP_, KS = DP / 16, DB = (DP + 31) / 32, PITCH = DP <= 32 ? 64 : DP <= 64 ? 128 : DP <= 96 && !WHOLE ? 192 : 256, PIECES = PITCH / 16;
    static constexpr int TILE = KEYS * PITCH, REQ = TILE / 1024, RPR = 1024 / PITCH;  // a tile of K or V: bytes, requests of a KB, whole rows per request
    // Where the second product's blocks of 32 columns are more than the head, a column of ones behind it in V makes the sums of the (rounded)
    // probabilities, which are a sixth of the vector instructions otherwise: 4096 queries, 4608 keys, 24 heads of 80 184 -> 171 us; 1157, 333 (all of them), 4 x 16 of 72
    // 23.4 -> 22.7
    static constexpr bool ONES = ONES_;
    static __host__ __device__ constexpr int fk(int row) { return PITCH == 256 ? row & 15 : PITCH == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
    static __host__ __device__ constexpr int fv(int row) { return PITCH == 256 ? 4 * (row & 3) : PITCH == 128 ? 4 * ((row >> 1) & 1) : 0; }
};

__device__ inline void copy16(uint32_t dst, const char *src, uint32_t off) {
    dst = __builtin_amdgcn_readfirstlane(dst);  // (the same in all lanes anyway)
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)src), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)src >> 32));
    const char *base = (const char *)(((uintptr_t)hi << 32) | lo);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
// zeros made on the spot: four registers that hold them through the whole loop are four too many
__device__ inline void clear16(uint32_t dst) {
    u32x4_t z;
    asm volatile("v_mov_b32 %0, 0\n\tv_mov_b32 %1, 0" : "=v"(z[0]), "=v"(z[1]));
    z[2] = z[0];
    z[3] = z[1];
    *(__attribute__((address_space(3))) u32x4_t *)dst = z;
}

// x of this lane and of the lane 32 further, in both
__device__ inline float across_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
    return __builtin_fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}
__device__ inline float across_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
    return bits_f32(r[0]) + bits_f32(r[1]);
}

// Running softmax and output of 32 rows: lane l holds row l % 32; of the output's block db element e is column 32 db + 8 (e / 4) + 4 (l / 32) + e % 4.
// Scores s of a step: block kb, element e is key 32 kb + 8 (e / 4) + 4 (l / 32) + e % 4.
template <bool BF16, typename H>
struct State {
    using E = Elem<BF16>;
    using vec = typename E::vec;
    float16_t o[H::DB];
    float top, sum;  // what the exponentials refer to, RAISED below the maximum in use, in units of log2; this lane's part of the sum
    __device__ inline void clear() {
#pragma unroll
        for (int d = 0; d < H::DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.f;
        top = -__builtin_huge_valf();
        sum = 0.f;
    }
    // keys without a bit get a score of minus infinity
    template <int NB>
    static __device__ inline void mask(float16_t (&s)[NB], uint64_t bits, int lane) {
        if (bits == ~0ull >> (64 - 32 * NB)) return;
#pragma unroll
        for (int kb = 0; kb < NB; kb++) {
            const uint32_t w = (uint32_t)(bits >> (32 * kb)) >> (4 * (lane >> 5));
#pragma unroll
            for (int e = 0; e < 16; e++) {  // (the bit over the whole word picks the score or minus infinity: two instructions)
                const uint32_t in = (uint32_t)__builtin_amdgcn_sbfe((int)w, 8 * (e >> 2) + (e & 3), 1);
                s[kb][e] = bits_f32((f32_bits(s[kb][e]) & in) | (0xFF800000u & ~in));
            }
        }
    }
    template <int NB>
    static __device__ inline float highest(const float16_t (&s)[NB]) {
        float m[2 * NB];  // (as many chains: a vector instruction waits for the one before it)
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            m[i] = s[i >> 1][8 * (i & 1)];
#pragma unroll
            for (int e = 1; e < 8; e++) m[i] = __builtin_fmaxf(m[i], s[i >> 1][8 * (i & 1) + e]);
        }
        float top = __builtin_fmaxf(m[0], m[1]);
        if constexpr (NB == 2) top = __builtin_fmaxf(top, __builtin_fmaxf(m[2], m[3]));
        return across_max(top);
    }
    // A new maximum of a row (of scores; times scale2, in units of log2).  The one in use only has to keep the exponentials in range: it moves when a
    // row's is more than 2^8 times off, so that the outputs are rarely scaled.  How far off goes by the exponentials' own fma, rounded once: around
    // 2^27 neighbours in fp32 are 8 to 16 apart, where a rounded maximum compared with a rounded sum let an fp16 probability of 2^16 through, an
    // infinity.  The maximum in use is a rounded number, too, half such a distance off, so that fp16 is in range for scores below 2^28, bf16 2^31.
    __device__ inline void raise(float high, float scale2) {
        if (__any(__builtin_fmaf(high, scale2, -top) > E::RAISED + 8.f)) {
            const float m = high * scale2 - E::RAISED, now = m > top ? m : top;
            const float f = top == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= f;
#pragma unroll
            for (int d = 0; d < H::DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= f;
        }
    }
    // left operands of v^T p for 16 keys from row 16 n of the values in LDS on
    static __device__ inline void read_v(vec (&vf)[H::DB], const char *v, int n, int lane) {
        const int g = lane >> 4, i = lane & 15, h = lane >> 5;
        const char *vrow = v + (4 * h + (i >> 2)) * H::PITCH + (i & 1) * 8;
        const int piece = (g & 1) * 2 + ((i >> 1) & 1), f = H::fv(i >> 2);
        typedef short short4_t __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) short4_t *lds_t;
#pragma unroll
        for (int d = 0; d < H::DB; d++) {
            const char *at = vrow + 16 * n * H::PITCH + ((4 * d + piece) ^ f) * 16;
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(at + 8 * H::PITCH));
            vf[d] = __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    // the right operand: probabilities of 16 keys, rounded
    template <int NB, bool ONES>
    __device__ inline vec exponentials(const float16_t (&s)[NB], int n, float scale2, float ref) {
        float x[8];
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n >> 1][8 * (n & 1) + e], scale2, -ref));
        if (!ONES) sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = E::pair(x[2 * e], x[2 * e + 1]);
        return __builtin_bit_cast(vec, w);
    }
    __device__ inline float reference() const { return top == -__builtin_huge_valf() ? 0.f : top; }
    // A step's scores and values (v in LDS) join the sums, 16 keys at a time: while the matrix cores multiply the probabilities of
    // one 16, those of the next are made and the operands of the one behind it are on their way.
    template <bool ONES, int NB>
    __device__ inline void attend(float16_t (&s)[NB], uint64_t bits, float scale2, const char *v, int lane) {
        vec vf[2][H::DB], pr[2];
        read_v(vf[0], v, 0, lane);
        mask(s, bits, lane);
        raise(highest(s), scale2);
        const float ref = reference();
        pr[0] = exponentials<NB, ONES>(s, 0, scale2, ref);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 2 * NB; n++) {
            if (n < 2 * NB - 1) {
                read_v(vf[(n + 1) & 1], v, n + 1, lane);
                pr[(n + 1) & 1] = exponentials<NB, ONES>(s, n + 1, scale2, ref);
            }
#pragma unroll
            for (int d = 0; d < H::DB; d++) o[d] = E::mfma(vf[n & 1][d], pr[n & 1], o[d]);
            if (n < 2 * NB - 1) {
#pragma unroll
                for (int d = 0; d < H::DB; d++) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 20 / H::DB, 0);
                    __builtin_amdgcn_sched_group_barrier(0x400, 8 / H::DB, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// Sixteen columns from c0 on of this lane's row of the output: the lane has c0 + 4 (lane / 32) + [0, 4) in x[0 .. 3] and the same 8 further in
// x[4 .. 7].  The half-waves exchange, so that each has 8 in a row and stores 16 bytes.
template <bool BF16>
__device__ inline void store_columns(char *out, const float (&x)[8], float r, int c0, int columns, int lane) {
    const int h = lane >> 5;
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t lo = Elem<BF16>::pair(x[2 * j] * r, x[2 * j + 1] * r), hi = Elem<BF16>::pair(x[4 + 2 * j] * r, x[5 + 2 * j] * r);
        const uint32_t give = h ? lo : hi, got = (uint32_t)__shfl_xor((int)give, 32);
        w[j] = h ? got : lo;
        w[2 + j] = h ? hi : got;
    }
    const int c = c0 + 8 * h;
    if (c < columns) *(u32x4_t *)(out + c * 2) = w;
}
__device__ inline float inverse(float sum) { return sum > 0.f ? 1.0f / sum : sum == 0.f ? 0.f : sum; }  // (a NaN stays one)

// Pieces from `first` to the last that is multiplied, of ROWS rows of K in LDS (stages one behind the other): zeros
template <typename H, int ROWS>
__device__ inline void zero_columns(char *lds, int first, int thread, int threads) {
    for (int r = thread; r < ROWS; r += threads)
        for (int c = first; c < H::DP / 8; c++) *(u32x4_t *)(lds + r * H::PITCH + (c ^ H::fk(r % KEYS)) * 16) = u32x4_t{0, 0, 0, 0};
}

// The copies of K and V to LDS by the WAVES waves of a workgroup: stages 0 and 1 of K, then those of V.
template <typename H, int WAVES>
struct Copies {
    // Request i of a wave brings rows row0 + i * RPR.  What a lane reads of them: V the same piece every time, K piece c ^ 4 i (f's
    // two steps: the wave's rows start on a multiple of 16 where there are four requests, of 8 where there are two).  With 12 pieces in a
    // row a request is five rows and a third: each has its own rows, pieces and offsets.
    static constexpr bool EVEN = H::PITCH != 192;
    static constexpr int REQ = H::REQ / WAVES > 0 ? H::REQ / WAVES : 1, ACTIVE = H::REQ / REQ;  // per wave; waves that make any
    static_assert(!EVEN || REQ == 1 || (REQ * H::RPR <= 16 && H::fk(H::RPR) == 4 && H::fv(H::RPR) == 0), "");
    static_assert(EVEN || (H::REQ % WAVES == 0 && H::fv(1) == 0 && H::fk(15) < 4), "");
    static constexpr int OWN = EVEN ? 1 : REQ;
    const char *kp, *vp;
    long long k_token, v_token;
    uint32_t dst, ok[OWN], ov[OWN], ck[OWN];
    int row[OWN], count, bytes;
    bool any, in_row[OWN];  // (whether V's piece lies in the head)
    // keys and values of a head from the first one on, the bytes from one to the next, channels of a head, how many there are, 1 in the tensors' type
    __device__ inline Copies(char *lds, const char *k_, const char *v_, long long k_token_, long long v_token_, int D, int count_, int wave, int lane, uint32_t one) {
        kp = k_;
        vp = v_;
        k_token = k_token_;
        v_token = v_token_;
        count = count_;
        bytes = D * 2;
        any = wave < ACTIVE;
        dst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + wave * REQ * 1024;
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const int piece = (wave * REQ + i) * 64 + lane, place = piece % H::PIECES;
            row[i] = piece / H::PIECES;
            ck[i] = (place ^ H::fk(row[i])) * 16;
            ok[i] = (uint32_t)(row[i] * k_token);
            ov[i] = (uint32_t)(row[i] * v_token) + (place ^ H::fv(row[i])) * 16;
            in_row[i] = (place ^ H::fv(row[i])) * 16 < bytes;
            if (!EVEN) ok[i] += ck[i];
        }
        // columns behind the head's end, as far as they are multiplied, are zero in K for good: no copy writes there (all waves see it behind the
        // first step's barrier)
        zero_columns<H, 2 * KEYS>(lds, D / 8, threadIdx.x, WAVES * 64);
        if constexpr (H::ONES) {
            for (int r = threadIdx.x; r < 2 * KEYS; r += WAVES * 64)
                *(u32x4_t *)(lds + 2 * H::TILE + r * H::PITCH + ((D / 8) ^ H::fv(r)) * 16) = u32x4_t{one, 0, 0, 0};
        }
    }
    // K of step `step` to stage `slot`.  Rows behind the last key are not read: their scores are masked whatever they are.
    __device__ __forceinline__ void k(int step, int slot) {
        if (!any) return;
        const char *k = kp + (long long)step * KEYS * k_token;
        const int left = count - step * KEYS;
        if constexpr (EVEN) {
            uint32_t c0 = ck[0];
            asm volatile("" : "+v"(c0));  // (what differs between the requests is worked out anew: registers are short)
            if (left >= KEYS && bytes == H::PITCH) {
#pragma unroll
                for (int i = 0; i < REQ; i++) copy16(dst + slot * H::TILE + i * 1024, k + i * H::RPR * k_token, ok[0] + (c0 ^ (64 * i)));
            } else {
#pragma unroll
                for (int i = 0; i < REQ; i++) {
                    const uint32_t c = c0 ^ (64 * i);
                    if ((int)c < bytes && row[0] < left - i * H::RPR) copy16(dst + slot * H::TILE + i * 1024, k + i * H::RPR * k_token, ok[0] + c);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < REQ; i++)
                if ((int)ck[i] < bytes && row[i] < left) copy16(dst + slot * H::TILE + i * 1024, k, ok[i]);
        }
    }
    // V: zeros for keys that do not count, since nothing times a NaN is one
    __device__ __forceinline__ void v(int step, int slot, uint64_t bits) {
        if (!any) return;
        const char *v = vp + (long long)step * KEYS * v_token;
        const uint32_t to = dst + (2 + slot) * H::TILE;
        if constexpr (EVEN) {
            if (!in_row[0]) return;
            if (bits == ~0ull) {
#pragma unroll
                for (int i = 0; i < REQ; i++) copy16(to + i * 1024, v + i * H::RPR * v_token, ov[0]);
            } else {
#pragma unroll
                for (int i = 0; i < REQ; i++) {
                    if ((bits >> (i * H::RPR)) >> row[0] & 1) copy16(to + i * 1024, v + i * H::RPR * v_token, ov[0]);
                    else clear16(to + i * 1024 + (threadIdx.x & 63) * 16);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < REQ; i++) {
                if (!in_row[i]) continue;
                if (bits == ~0ull || (bits >> row[i] & 1)) copy16(to + i * 1024, v, ov[i]);
                else clear16(to + i * 1024 + (threadIdx.x & 63) * 16);
            }
        }
    }
};

}  // namespace attention
}  // namespace svdq
