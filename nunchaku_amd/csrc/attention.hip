// Softmax attention of queries to the keys of an encoder: out[b][t][h] = sum_j p_j v[b][j][h / G], p = softmax over the valid keys j
// of scale * q[b][t][h] . k[b][j][h / G]; zero where no key is valid.  G = heads / kv_heads query heads share a head of keys and
// values: a "row" below is one (token, head of the group) pair, row r = t * G + g of key head h / G.
//
// One pass over the keys, 64 at a time, with the running maximum and sum of the softmax in fp32.  The scores are formed as K q^T on
// v_mfma_f32_32x32x16: a lane then holds 32 keys' scores of ONE row (the other 32 are 32 lanes away), so the maximum and the sum
// take one exchange between lanes, and the scores, rounded to the inputs' type, are the right operand of v^T p^T as they are: the
// instruction contracts 8 keys per lane, which 8 is free, as long as the left operand holds the same.  That operand is v down the
// columns, which LDS reads that transpose 4 x 16 blocks (ds_read_b64_tr_b16) make of plain rows.
// The probabilities are rounded to the inputs' type for that product (half a step relative each, like the result), sums stay in fp32: of the
// probabilities as they are, or of the rounded ones where the product makes them (then both sides of the division have the same roundings: relative
// errors of 0.00226 instead of 0.00234 in bf16, 0.000278 instead of 0.000289 in fp16, for normal scores and values).
//
// Rows of K and V in LDS: pieces of 16 bytes, piece c of row r at place c ^ f(r), so that neither 16 lanes that read one piece of 16
// rows (K) nor 32 lanes that read 64 bytes of 4 rows (V) meet in a bank.  What no key stands for (rows behind the last key, masked
// ones) is not read from V at all, whatever it holds: zeros stand there.
#include "svdq_common.h"

using namespace svdq;

namespace {

struct AttentionParams {
    const char *q, *k, *v;
    char *out;
    const int *key_lengths, *cu_seqlens;
    const uint8_t *mask;
    float *partial;                                // keys-split form with several parts: [part][b][hkv][rows] x D, then {maximum, sum} pairs
    long long qs[3], ks[3], vs[3], os[3], mask_b;  // bytes: batch, token, head
    int B, Hkv, G, D, Tq, Tk, rows, row_blocks, parts, spread;
    float scale2;  // scale * log2(e)
};

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

// The keys of batch entry b: the first one's row in the tensors (packed sequences) and how many there are.
__device__ inline void keys_of(const AttentionParams &p, int b, long long &first, int &count) {
    first = 0;
    count = p.Tk;
    if (p.cu_seqlens) {  // (offsets that are not in order or beyond the end give fewer keys, never others)
        int lo = p.cu_seqlens[b], hi = p.cu_seqlens[b + 1];
        lo = lo < 0 ? 0 : lo > p.Tk ? p.Tk : lo;
        hi = hi < lo ? lo : hi > p.Tk ? p.Tk : hi;
        first = __builtin_amdgcn_readfirstlane(lo);
        count = hi - lo;
    } else if (p.key_lengths) {
        const int n = p.key_lengths[b];
        count = n < 0 ? 0 : n < p.Tk ? n : p.Tk;
    }
    count = __builtin_amdgcn_readfirstlane(count);
}

// The steps of SIZE keys that hold any, in order, with a bit for every key that counts.  With a mask the bytes of the step behind the
// next one are on their way while a step is worked on; steps without a key are left out.
template <bool MASK, int SIZE = KEYS>
struct Steps {
    const uint8_t *mask;
    int count, steps, stride, at, lane;  // at: the next candidate
    uint32_t byte;
    uint64_t bits;  // of the step that next() returned
    __device__ inline void fetch() {
        if (MASK) {
            const int key = at * SIZE + lane;
            byte = 0;
            if (lane < SIZE && key < count) byte = mask[key];
        }
    }
    __device__ inline void start(const uint8_t *m, int count_, int first, int end, int stride_, int lane_) {
        mask = m;
        count = count_;
        steps = end;
        stride = stride_;
        at = first;
        lane = lane_;
        byte = 0;
        if (at < steps) fetch();
    }
    // the next step with a key, or -1
    __device__ inline int next() {
        while (at < steps) {
            const int step = at, left = count - step * SIZE;
            bits = MASK ? __ballot(byte != 0) : left >= SIZE ? ~0ull >> (64 - SIZE) : (1ull << left) - 1;
            at += stride;
            if (at < steps) fetch();
            if (!MASK || bits) return step;
        }
        bits = 0;
        return -1;
    }
};

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

// This lane's row of queries as the right operand: elements 16 ks + 8 (lane / 32) ... + 7
template <bool BF16, typename H>
__device__ inline void load_q(const AttentionParams &p, typename Elem<BF16>::vec (&qf)[H::KS], int b, int hk, int row, int lane) {
    const int t = row / p.G, gq = row - t * p.G;
    const char *q = p.q + b * p.qs[0] + t * p.qs[1] + (long long)(hk * p.G + gq) * p.qs[2];
#pragma unroll
    for (int ks = 0; ks < H::KS; ks++) {
        const int c = 16 * ks + 8 * (lane >> 5);
        u32x4_t w = u32x4_t{0, 0, 0, 0};
        if (row < p.rows && c < p.D) w = *(const u32x4_t *)(q + c * 2);
        qf[ks] = __builtin_bit_cast(typename Elem<BF16>::vec, w);
    }
}

// The compiler waits for these loads where they are first used.  In the loop over the keys that wait would be for the copies that a step
// has just asked for, too, and at every step: this, in front of the loop and behind the first copies, is where they are waited for.
template <bool BF16, typename H>
__device__ inline void wait_for_q(typename Elem<BF16>::vec (&qf)[H::KS]) {
#pragma unroll
    for (int ks = 0; ks < H::KS; ks++) asm volatile("" : "+v"(qf[ks]));
}

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
__device__ inline char *row_of(const AttentionParams &p, int b, int hk, int row) {
    const int t = row / p.G, gq = row - t * p.G;
    return p.out + b * p.os[0] + t * p.os[1] + (long long)(hk * p.G + gq) * p.os[2];
}

// With the keys in parts: which one a workgroup has (taken out of its group), and its share of the steps 0 .. end
__device__ inline int take_part(const AttentionParams &p, int &group) {
    if (p.parts == 1) return 0;
    const int whole = group / p.parts, part = group - whole * p.parts;
    group = whole;
    return part;
}
__device__ inline void share(const AttentionParams &p, int part, int &begin, int &end) {
    if (p.parts == 1) return;
    const int each = end / p.parts, more = end - each * p.parts;
    begin = part * each + (part < more ? part : more);
    end = begin + each + (part < more);
}
// Where a part's share of a row goes, [part][b][hkv][row] x D, and its maximum and sum behind all of those
__device__ inline long long part_index(const AttentionParams &p, int part, int b, int hk, int row) {
    return (((long long)part * p.B + b) * p.Hkv + hk) * p.rows + row;
}
__device__ inline float *part_of(const AttentionParams &p, int part, int b, int hk, int row) { return p.partial + part_index(p, part, b, hk, row) * p.D; }
__device__ inline void store_stats(const AttentionParams &p, int part, int b, int hk, int row, float top, float sum) {
    float *ms = p.partial + (long long)p.parts * p.B * p.Hkv * p.rows * p.D + part_index(p, part, b, hk, row) * 2;
    ms[0] = top;
    ms[1] = sum;
}

// Which (row block, group) a workgroup takes, false: none.  A group's row blocks read the same keys (of a head, or of a part of its keys).
// Workgroups go round robin over 8 XCDs, each with an L2 of its own.  The row blocks of a group go to one XCD, the groups in turn over
// the XCDs (`spread`: a batch entry's keys may be many or few, and eight entries on an XCD each would leave some of them idle), or, where
// there are too few groups for that to come out even, an XCD gets a contiguous run of all row blocks.
__device__ inline bool block_of(const AttentionParams &p, int groups, int &rb, int &group) {
    const int id = blockIdx.x, xcd = id & 7, j = id >> 3;
    if (p.spread) {
        group = j / p.row_blocks * 8 + xcd;
        rb = j % p.row_blocks;
        return group < groups;
    }
    const int total = groups * p.row_blocks, per = total >> 3, more = total & 7;
    const int at = xcd * per + (xcd < more ? xcd : more) + j;
    rb = at % p.row_blocks;
    group = at / p.row_blocks;
    return true;
}

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
    __device__ inline Copies(const AttentionParams &p, char *lds, int b, int hk, long long first, int count_, int wave, int lane, uint32_t one) {
        kp = p.k + b * p.ks[0] * (p.cu_seqlens ? 0 : 1) + first * p.ks[1] + hk * p.ks[2];
        vp = p.v + b * p.vs[0] * (p.cu_seqlens ? 0 : 1) + first * p.vs[1] + hk * p.vs[2];
        k_token = p.ks[1];
        v_token = p.vs[1];
        count = count_;
        bytes = p.D * 2;
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
        zero_columns<H, 2 * KEYS>(lds, p.D / 8, threadIdx.x, WAVES * 64);
        if constexpr (H::ONES) {
            for (int r = threadIdx.x; r < 2 * KEYS; r += WAVES * 64)
                *(u32x4_t *)(lds + 2 * H::TILE + r * H::PITCH + ((p.D / 8) ^ H::fv(r)) * 16) = u32x4_t{one, 0, 0, 0};
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

// ---- rows form: 128 rows per workgroup, 32 per wave; all waves share the keys through LDS, two steps of them -------------------
// Bound by each wave's chain of scores, maximum, exponentials and second product: 4096 queries, 4573 keys, 24 heads of 128 in fp16 take 247 us,
// 931 TFLOP/s, the matrix cores busy 46 % of the cycles.  A step takes a workgroup by itself 1.12 us, each of two on a compute unit 1.08: the second wave
// of a SIMD hardly fills what the first leaves.  Short keys are first loads and stores besides: 1024 queries, 300 keys, 8 x 32 heads of 64 34 us.
template <bool BF16, int DP, bool MASK, bool ONES>
__global__ void __launch_bounds__(256, 2) attention_rows_kernel(AttentionParams p) {
    using H = Head<DP, false, ONES>;
    using E = Elem<BF16>;
    using vec = typename E::vec;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    int rb, group;
    if (!block_of(p, p.Hkv * p.B * p.parts, rb, group)) return;
    const int part = take_part(p, group), hk = group % p.Hkv, b = group / p.Hkv;
    long long first;
    int count;
    keys_of(p, b, first, count);
    const int row = (rb * 4 + wave) * 32 + col;
    vec qf[H::KS];
    State<BF16, H> st;
    load_q<BF16, H>(p, qf, b, hk, row, lane);
    st.clear();
    Copies<H, 4> copies(p, lds, b, hk, first, count, wave, lane, E::ONE);
    Steps<MASK> list;
    int begin = 0, end = (count + KEYS - 1) / KEYS;
    share(p, part, begin, end);
    list.start(MASK ? p.mask + b * p.mask_b : nullptr, count, begin, end, 1, lane);
    int step = list.next();
    uint64_t bits = list.bits;
    if (step >= 0) {
        copies.k(step, 0);
        copies.v(step, 0, bits);
    }
    wait_for_q<BF16, H>(qf);
    for (int slot = 0; step >= 0; slot ^= 1) {
        // K and V of this step have landed, of all waves, and nobody reads what the next requests overwrite
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int next = list.next();
        if (next >= 0) {
            copies.k(next, slot ^ 1);
            copies.v(next, slot ^ 1, list.bits);
        }
        const char *k = lds + slot * H::TILE + col * H::PITCH, *v = lds + (2 + slot) * H::TILE;
        float16_t s[2];
        // operands of four matrix instructions at a time, the next four's on their way
        constexpr int N = 2 * H::KS, GROUP = N % 4 == 0 ? 4 : 2;
        vec kf[2][GROUP];
        auto read_k = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < GROUP; i++) {
                const int n = g * GROUP + i, kb = n & 1, ks = n >> 1;
                kf[g & 1][i] = __builtin_bit_cast(vec, *(const u32x4_t *)(k + kb * 32 * H::PITCH + ((2 * ks + h) ^ H::fk(col)) * 16));
            }
        };
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[kb][e] = 0.f;
        read_k(0);
#pragma unroll
        for (int g = 0; g < N / GROUP; g++) {
            if (g + 1 < N / GROUP) read_k(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < GROUP; i++) {
                const int n = g * GROUP + i, kb = n & 1, ks = n >> 1;
                s[kb] = E::mfma(kf[g & 1][i], qf[ks], s[kb]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        st.template attend<H::ONES>(s, bits, p.scale2, v, lane);
        step = next;
        bits = list.bits;
    }
    if constexpr (H::ONES) {
#pragma unroll
        for (int g = 0; g < 4 * H::DB; g++)
            if (8 * g == p.D && h == 0) st.sum = st.o[g >> 2][4 * (g & 3)];
    }
    const float sum = across_sum(st.sum);
    if (p.parts > 1) {
        if (row >= p.rows) return;
        float *dst = part_of(p, part, b, hk, row);
#pragma unroll
        for (int d = 0; d < H::DB; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int c = 32 * d + 8 * g + 4 * h;
                if (c < p.D) *(float4_t *)(dst + c) = float4_t{st.o[d][4 * g], st.o[d][4 * g + 1], st.o[d][4 * g + 2], st.o[d][4 * g + 3]};
            }
        if (h == 0) store_stats(p, part, b, hk, row, st.top, sum);
        return;
    }
    const float r = inverse(sum);
    char *out = row_of(p, b, hk, row);
#pragma unroll
    for (int u = 0; u < 2 * H::DB; u++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = st.o[u >> 1][8 * (u & 1) + e];
        store_columns<BF16>(out, x, r, 16 * u, row < p.rows ? p.D : 0, lane);
    }
}

// ---- keys form: 32 rows per workgroup, whose waves take every fourth step (of 32 keys) of the part's keys, each through its own LDS, a
// step ahead, and meet in LDS at the end; the parts of a row block meet in attention_join_kernel ------------------------------------
// Bound by K's and V's way from memory: single tokens of 8 sequences of up to 4096 keys, 32 heads over 8 of 128: 24 us
// with the join's 4; all of 8192 48 us, 5.5 TB/s.
template <bool BF16, int DP, bool MASK>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1) attention_keys_kernel(AttentionParams p) {
    using H = Head<DP, true>;
    using E = Elem<BF16>;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    int rb, group;
    if (!block_of(p, p.Hkv * p.B * p.parts, rb, group)) return;
    const int part = take_part(p, group), hk = group % p.Hkv, b = group / p.Hkv;
    long long first;
    int count;
    keys_of(p, b, first, count);
    const int row = rb * 32 + col;
    typename E::vec qf[H::KS];
    load_q<BF16, H>(p, qf, b, hk, row, lane);
    const char *kp = p.k + b * p.ks[0] * (p.cu_seqlens ? 0 : 1) + first * p.ks[1] + hk * p.ks[2];
    const char *vp = p.v + b * p.vs[0] * (p.cu_seqlens ? 0 : 1) + first * p.vs[1] + hk * p.vs[2];
    constexpr int SIZE = 32, REQ = H::REQ / 2, STAGE = H::TILE;  // a stage: 32 rows of K, then of V
    char *mine = lds + wave * 2 * STAGE;
    const uint32_t area = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + wave * 2 * STAGE;
    const int bytes = p.D * 2;
    int begin = 0, end = (count + SIZE - 1) / SIZE;
    share(p, part, begin, end);
    // Request i brings rows r0 + i * RPR: of V the same piece every time, of K the pieces that f has there
    const int r0 = lane / H::PIECES, ck = ((lane % H::PIECES) ^ H::fk(r0)) * 16, cv = ((lane % H::PIECES) ^ H::fv(r0)) * 16;
    const uint32_t ok = (uint32_t)(r0 * p.ks[1]), ov = (uint32_t)(r0 * p.vs[1]) + cv;
    static_assert(H::fv(H::RPR) == 0 && (H::RPR == 16 || H::fk(H::RPR) == 4), "");
    // columns behind the head's end are zero in K for good (the wait for a step's copies is one for these, too)
    zero_columns<H, SIZE>(mine, p.D / 8, lane, 64);
    zero_columns<H, SIZE>(mine + STAGE, p.D / 8, lane, 64);
    auto request = [&](int step, int slot, uint64_t bits) __attribute__((always_inline)) {
        const char *k = kp + (long long)step * SIZE * p.ks[1], *v = vp + (long long)step * SIZE * p.vs[1];
        const int left = count - step * SIZE;
        const uint32_t dst = area + slot * STAGE;
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            const int c = ck ^ (64 * (i & (16 / H::RPR - 1)));
            if (c < bytes && r0 < left - i * H::RPR) copy16(dst + i * 1024, k + i * H::RPR * p.ks[1], ok + c);
        }
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            if (cv >= bytes) continue;
            if ((bits >> (i * H::RPR)) >> r0 & 1) copy16(dst + STAGE / 2 + i * 1024, v + i * H::RPR * p.vs[1], ov);
            else clear16(dst + STAGE / 2 + i * 1024 + lane * 16);
        }
    };
    State<BF16, H> st;
    st.clear();
    Steps<MASK, SIZE> list;
    list.start(MASK ? p.mask + b * p.mask_b : nullptr, count, begin + wave, end, 4, lane);
    int step = list.next();
    uint64_t bits = list.bits;
    if (step >= 0) request(step, 0, bits);
    wait_for_q<BF16, H>(qf);
    for (int slot = 0; step >= 0; slot ^= 1) {
        const int next = list.next();
        if (next >= 0) request(next, slot ^ 1, list.bits);
        // This step's copies have landed when no more than the next one's are on their way.  Of a step with keys that do not count some
        // requests may have had no lane to make them: then all have to land.
        if (next >= 0 && list.bits == 0xFFFFFFFFull) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * REQ) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        const char *k = mine + slot * STAGE + col * H::PITCH;
        float16_t s[1];
#pragma unroll
        for (int e = 0; e < 16; e++) s[0][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < H::KS; ks++) {
            const u32x4_t w = *(const u32x4_t *)(k + ((2 * ks + h) ^ H::fk(col)) * 16);
            s[0] = E::mfma(__builtin_bit_cast(typename E::vec, w), qf[ks], s[0]);
        }
        st.template attend<false>(s, bits, p.scale2, mine + slot * STAGE + STAGE / 2, lane);
        step = next;
        bits = list.bits;
    }
    // The waves meet.  Each leaves its maximum, sum and outputs in the place of its own stages, 16 columns (a unit) of 64 lanes in 2 KB, and takes
    // every fourth unit of all four, scaled to the highest maximum.  (All sums in one wave's registers: single tokens, 40 keys, D = 128 8.2 us
    // against 6.1.)
    constexpr int UNITS = 2 * H::DB, AREA = 2 * STAGE;
    static_assert(256 + UNITS * 2048 <= AREA, "");
    const float own = across_sum(st.sum);
    if (h == 0) {
        ((float *)mine)[col] = st.top;
        ((float *)mine)[32 + col] = own;
    }
    if (row < p.rows) {
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int d = u >> 1, e = 8 * (u & 1) + 4 * i;
                ((float4_t *)(mine + 256 + u * 2048 + i * 1024))[lane] = float4_t{st.o[d][e], st.o[d][e + 1], st.o[d][e + 2], st.o[d][e + 3]};
            }
    }
    __syncthreads();
    float top = -__builtin_huge_valf(), sum = 0.f, f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) top = __builtin_fmaxf(top, ((float *)(lds + i * AREA))[col]);
    const float ref = top == -__builtin_huge_valf() ? 0.f : top;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[i] = __builtin_amdgcn_exp2f(((float *)(lds + i * AREA))[col] - ref);
        sum += ((float *)(lds + i * AREA))[32 + col] * f[i];
    }
    const float r = inverse(sum);
    char *out = row_of(p, b, hk, row);
    float *dst = part_of(p, part, b, hk, row);
    const int columns = row < p.rows ? p.D : 0;
    for (int u = wave; u < UNITS; u += 4) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float4_t y = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float4_t o = ((float4_t *)(lds + w * AREA + 256 + u * 2048 + i * 1024))[lane];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(o[e], f[w], y[e]);
            }
            const int c = 16 * u + 8 * i + 4 * h;
            if (p.parts > 1 && c < columns) *(float4_t *)(dst + c) = y;
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * i + e] = y[e];
        }
        if (p.parts == 1) store_columns<BF16>(out, x, r, 16 * u, columns, lane);
    }
    if (p.parts > 1 && wave == 0 && h == 0 && row < p.rows) store_stats(p, part, b, hk, row, top, sum);
}

// Adds the parts of every row (at most 64): four waves a workgroup, PER of them to a row, two columns per lane; a wave takes every PER-th part, all
// requested at once.  Lane i of every wave holds part i's share of the row.
constexpr int MAX_PARTS = 64;
template <bool BF16, int PER>
__global__ void __launch_bounds__(256) attention_join_kernel(AttentionParams p) {
    constexpr int MOST = 16;  // parts a wave
    __shared__ float sums[PER == 1 ? 1 : 4][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = wave % PER;
    const long long all = (long long)p.B * p.Hkv * p.rows, at = (long long)blockIdx.x * (4 / PER) + wave / PER;
    if (PER == 1 && at >= all) return;
    const float *ms = p.partial + p.parts * all * p.D;
    const int c = lane * 2 < p.D ? lane * 2 : 0;
    typedef float float2_t __attribute__((ext_vector_type(2)));
    float2_t part[MOST];
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        part[i] = float2_t{0.f, 0.f};
        if (sub + PER * i < p.parts) part[i] = *(const float2_t *)(p.partial + ((sub + PER * i) * all + at) * p.D + c);
    }
    float top = -__builtin_huge_valf(), sum = 0.f;
    if (lane < p.parts) {
        const float2_t t = *(const float2_t *)(ms + (lane * all + at) * 2);
        top = t[0];
        sum = t[1];
    }
    float most = top;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, d));
    const float f = __builtin_amdgcn_exp2f(top - (most == -__builtin_huge_valf() ? 0.f : most));
    sum *= f;
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < MOST; i++) {  // (zero times zero behind the last part)
        const float g = bits_f32(__builtin_amdgcn_readlane(f32_bits(f), sub + PER * i));
        x = __builtin_fmaf(part[i][0], g, x);
        y = __builtin_fmaf(part[i][1], g, y);
    }
    if constexpr (PER > 1) {
        sums[wave][0][lane] = x;
        sums[wave][1][lane] = y;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int i = 1; i < 4; i++) {
            x += sums[i][0][lane];
            y += sums[i][1][lane];
        }
    }
    if (lane * 2 >= p.D) return;
    const float r = inverse(sum);
    const int bh = (int)(at / p.rows), row = (int)(at - (long long)bh * p.rows), b = bh / p.Hkv, hk = bh - b * p.Hkv;
    *(uint32_t *)(row_of(p, b, hk, row) + c * 2) = Elem<BF16>::pair(x * r, y * r);
}

template <bool BF16, int DP, bool MASK, bool ONES>
int launch_kernels(const AttentionParams &p, bool keys, hipStream_t st) {
    const int lds = keys ? 8 * Head<DP, true>::TILE : 4 * Head<DP>::TILE;
    static bool reserved[2][64] = {{false}};
    const void *kernel = keys ? (const void *)attention_keys_kernel<BF16, DP, MASK> : (const void *)attention_rows_kernel<BF16, DP, MASK, ONES>;
    if (int rc = reserve_lds(kernel, lds, reserved[keys], "cross_attention")) return rc;
    const long long groups = (long long)p.parts * p.Hkv * p.B;
    const dim3 grid((unsigned)((p.spread ? (groups + 7) / 8 * 8 : groups) * p.row_blocks)), block(256);
    if (keys) SVDQ_LAUNCH((attention_keys_kernel<BF16, DP, MASK>), grid, block, lds, st, p);
    else SVDQ_LAUNCH((attention_rows_kernel<BF16, DP, MASK, ONES>), grid, block, lds, st, p);
    int rc = check_launch("cross_attention");
    if (rc || p.parts == 1) return rc;
    const long long all = (long long)p.B * p.Hkv * p.rows;
    // One wave a row where rows are many (8 heads of 128, 1024 queries in four parts 41.5 -> 36.4 us, 2 of 64, 4000 queries 32.6 -> 27.2), four where they are
    // few (2 x 8 heads of 64, single tokens in 16 parts 8.3 -> 8.0) or the parts more than one wave asks for at once
    if (p.parts <= 16 && all > 1024) SVDQ_LAUNCH((attention_join_kernel<BF16, 1>), dim3((unsigned)((all + 3) / 4)), dim3(256), 0, st, p);
    else SVDQ_LAUNCH((attention_join_kernel<BF16, 4>), dim3((unsigned)all), dim3(256), 0, st, p);
    return check_launch("cross_attention");
}

template <bool BF16, int DP, bool MASK>
int launch_head(const AttentionParams &p, bool keys, hipStream_t st) {
    if (p.D < 32 * Head<DP>::DB) return launch_kernels<BF16, DP, MASK, true>(p, keys, st);
    if constexpr (DP % 32 == 0) return launch_kernels<BF16, DP, MASK, false>(p, keys, st);
    return SVDQ_EUNSUPPORTED;  // (not reached: the blocks of 80 end at 96)
}
template <bool BF16, bool MASK>
int launch_heads(const AttentionParams &p, bool keys, hipStream_t st) {
    if (p.D <= 32) return launch_head<BF16, 32, MASK>(p, keys, st);
    if (p.D <= 64) return launch_head<BF16, 64, MASK>(p, keys, st);
    if (p.D <= 80) return launch_head<BF16, 80, MASK>(p, keys, st);
    if (p.D <= 96) return launch_head<BF16, 96, MASK>(p, keys, st);
    return launch_head<BF16, 128, MASK>(p, keys, st);
}

// Which form a call takes and how many parts it divides the keys into: the least time by a model of the busiest compute unit, us, whose constants are those
// of 192 shapes in both forms; of 240 shapes in both forms and 1 .. 32 parts what it chooses is 0.6 % behind the fastest on average, 15 % at most.  The rows form reads K and
// V once per 128 rows, the keys form has its waves side by side on one 32; parts of the keys fill the compute units and cost a join.  Chosen / the other form or no
// parts, us: 24 heads of 72, 1024 queries, 333 keys (768 blocks of 32) rows 11.9 / 25.0; 64 heads of 64, 130 queries, 1024 keys keys 13.6 / 18.0; 8 heads of 128, 512
// queries, 4096 keys rows in eight parts 26.6 / keys in two 34.6, rows whole 78; single tokens, 8 key heads of 128: 333 keys 9.1 / 9.3 in three, 512 9.5 in four / 10.5, 4096
// 9.9 in 32 / 49; 32 x 8 key heads of 64, 2048 keys 25.7 / 29.2 in two.
struct Plan {
    bool keys;
    long long row_blocks, parts, workspace;
};
struct Cost {
    int head_dim;                    // up to
    float rows_base, alone, share;   // rows form: launch, first and last; a step of 64 keys of a workgroup by itself, of each of several
    float keys_base, round;          // keys form: the same; a round of four waves' 32 keys
};
constexpr Cost costs[] = {{64, 3.7f, 0.84f, 0.63f, 4.3f, 0.8f}, {96, 3.9f, 1.03f, 0.85f, 5.0f, 1.3f}, {128, 5.2f, 1.12f, 1.08f, 5.4f, 1.4f}};

Plan plan_of(const svdq_cross_attention_args *a, int cus) {
    const long long rows = a->q_len * (a->heads / a->kv_heads), bh = a->batch * a->kv_heads;
    const long long keys_each = a->cu_seqlens_k ? (a->k_len + a->batch - 1) / a->batch : a->k_len;
    const long long blocks[2] = {(rows + 127) / 128 * bh, (rows + 31) / 32 * bh}, steps[2] = {(keys_each + KEYS - 1) / KEYS, (keys_each + 31) / 32};
    const Cost &c = a->head_dim <= 64 ? costs[0] : a->head_dim <= 96 ? costs[1] : costs[2];
    Plan plan = {true, 1, 1, 0};
    float best = 0.f;
    for (int keys = rows <= 32; keys < 2; keys++) {
        for (long long parts = 1; parts <= MAX_PARTS; parts++) {
            if (parts > 1 && (blocks[keys] * parts > (keys ? 1 : 2) * cus || steps[keys] < (keys ? 4 : 1) * (parts - 1))) break;
            float t;
            if (keys) {
                // two workgroups to a compute unit with heads up to 64, one with wider ones (LDS)
                const long long rounds = (steps[1] + 4 * parts - 1) / (4 * parts), slots = a->head_dim <= 64 ? 2 * cus : cus;
                t = (c.keys_base + (float)rounds * c.round * (blocks[1] * parts > cus && a->head_dim <= 64 ? 1.3f : 1.f)) * (float)((blocks[1] * parts + slots - 1) / slots);
            } else {
                const float each = (float)((blocks[0] * parts + cus - 1) / cus) * c.share;
                t = c.rows_base + (float)((steps[0] + parts - 1) / parts) * (each > c.alone ? each : c.alone);
            }
            if (parts > 1) t += 3.1f + (float)(bh * rows) * (float)(a->head_dim * 8 * parts) / 4.0e6f;  // the join, and the parts' way there and back
            if (best == 0.f || t < best) {
                best = t;
                plan.keys = keys;
                plan.parts = parts;
            }
        }
    }
    plan.row_blocks = plan.keys ? (rows + 31) / 32 : (rows + 127) / 128;
    plan.workspace = plan.parts > 1 ? plan.parts * bh * rows * (a->head_dim + 2) * 4 : 0;
    return plan;
}

int check_args(const svdq_cross_attention_args *a) {
    SVDQ_REQUIRE(a && a->q && a->k && a->v && a->out, "cross_attention: q, k, v and out must not be null");
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "cross_attention: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", (int)a->dtype);
    SVDQ_REQUIRE(a->batch > 0 && a->batch < 65536 && a->heads > 0 && a->heads < 65536 && a->kv_heads > 0 && a->heads % a->kv_heads == 0,
                 "cross_attention: batch (%lld) and heads (%lld) must be in 1..65535, kv_heads (%lld) must divide heads", (long long)a->batch, (long long)a->heads, (long long)a->kv_heads);
    SVDQ_REQUIRE(a->head_dim > 0 && a->head_dim <= 128 && a->head_dim % 8 == 0, "cross_attention: head_dim (%lld) must be a multiple of 8 up to 128", (long long)a->head_dim);
    SVDQ_REQUIRE(a->q_len > 0 && a->k_len > 0 && a->k_len < (1ll << 31) - 64, "cross_attention: q_len (%lld) and k_len (%lld) must be positive, k_len below 2^31 - 64", (long long)a->q_len,
                 (long long)a->k_len);
    SVDQ_REQUIRE(a->q_len < (1ll << 31) && a->q_len * (a->heads / a->kv_heads) < (1ll << 31) - 128,
                 "cross_attention: q_len (%lld) times the heads that share keys must be below 2^31 - 128", (long long)a->q_len);
    // (a launch takes fewer than 2^32 threads, 256 for 32 rows at most)
    const long long rows = a->q_len * (a->heads / a->kv_heads);
    SVDQ_REQUIRE((rows + 31) / 32 * (a->batch * a->kv_heads + 7) < (1ll << 24), "cross_attention: batch times kv_heads (%lld) groups of %lld rows of queries are too many for one launch",
                 (long long)(a->batch * a->kv_heads), rows);
    SVDQ_REQUIRE(!a->key_lengths + !a->key_mask + !a->cu_seqlens_k >= 2, "cross_attention: at most one of key_lengths, key_mask and cu_seqlens_k can be given");
    SVDQ_REQUIRE(a->scale > 0.f && a->scale < __builtin_huge_valf(), "cross_attention: scale must be a positive number");
    for (int i = 0; i < 3; i++)
        SVDQ_REQUIRE(a->q_stride[i] >= 0 && a->k_stride[i] >= 0 && a->v_stride[i] >= 0 && a->out_stride[i] >= 0 &&
                         (a->q_stride[i] | a->k_stride[i] | a->v_stride[i] | a->out_stride[i]) % 8 == 0,
                     "cross_attention: strides must be multiples of 8 elements (16 bytes)");
    SVDQ_REQUIRE(a->k_stride[1] < (1ll << 24) && a->v_stride[1] < (1ll << 24), "cross_attention: the tokens of k and v must be less than 2^24 elements apart");
    SVDQ_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)a->workspace) % 16 == 0, "cross_attention: pointers must be 16-byte aligned");
    SVDQ_REQUIRE(((uintptr_t)a->key_lengths | (uintptr_t)a->cu_seqlens_k) % 4 == 0, "cross_attention: key_lengths and cu_seqlens_k must be 4-byte aligned");
    return SVDQ_OK;
}

int current_compute_units(int &cus) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || (cus = compute_units(dev)) == 0) {
        (void)hipGetLastError();
        return fail(SVDQ_ELAUNCH, "cross_attention: no current device");
    }
    return SVDQ_OK;
}

}  // namespace

extern "C" int svdq_cross_attention_workspace(const svdq_cross_attention_args *a, int64_t *bytes) {
    if (int rc = check_args(a)) return rc;
    SVDQ_REQUIRE(bytes, "cross_attention: bytes must not be null");
    int cus;
    if (int rc = current_compute_units(cus)) return rc;
    *bytes = plan_of(a, cus).workspace;
    return SVDQ_OK;
}

extern "C" int svdq_cross_attention(const svdq_cross_attention_args *a, void *stream) {
    if (int rc = check_args(a)) return rc;
    int cus;
    if (int rc = current_compute_units(cus)) return rc;
    const Plan plan = plan_of(a, cus);
    SVDQ_REQUIRE(plan.workspace == 0 || (a->workspace && a->workspace_bytes >= plan.workspace), "cross_attention: needs a workspace of %lld bytes, got %lld", plan.workspace,
                 (long long)(a->workspace ? a->workspace_bytes : 0));
    AttentionParams p;
    p.q = (const char *)a->q;
    p.k = (const char *)a->k;
    p.v = (const char *)a->v;
    p.out = (char *)a->out;
    p.key_lengths = a->key_lengths;
    p.cu_seqlens = a->cu_seqlens_k;
    p.mask = (const uint8_t *)a->key_mask;
    p.partial = (float *)a->workspace;
    for (int i = 0; i < 3; i++) {
        p.qs[i] = a->q_stride[i] * 2;
        p.ks[i] = a->k_stride[i] * 2;
        p.vs[i] = a->v_stride[i] * 2;
        p.os[i] = a->out_stride[i] * 2;
    }
    p.mask_b = a->mask_stride;
    p.B = (int)a->batch;
    p.Hkv = (int)a->kv_heads;
    p.G = (int)(a->heads / a->kv_heads);
    p.D = (int)a->head_dim;
    p.Tq = (int)a->q_len;
    p.Tk = (int)a->k_len;
    p.rows = p.Tq * p.G;
    p.row_blocks = (int)plan.row_blocks;
    p.parts = (int)plan.parts;
    const long long groups = plan.parts * a->kv_heads * a->batch, turns = (groups + 7) / 8 * 8;
    p.spread = turns * 15 <= groups * 16;  // (at most a fifteenth more than an even share)
    p.scale2 = a->scale * 1.44269504088896340736f;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == SVDQ_BF16) return p.mask ? launch_heads<true, true>(p, plan.keys, st) : launch_heads<true, false>(p, plan.keys, st);
    return p.mask ? launch_heads<false, true>(p, plan.keys, st) : launch_heads<false, false>(p, plan.keys, st);
}
