// Softmax attention of the queries of several sequences to the keys of the same sequence, causal or not: query i of a sequence with n_q queries and
// n_k keys sees the keys j <= i + n_k - n_q (all of them where it is not causal).  G = heads / kv_heads query heads share a head of keys: a "row"
// below is one (token, head of the group) pair, row r = t * G + g of a sequence and a key head, so that a few tokens fill the rows of a matrix
// instruction, and the rows of a block end at nearly the same key.
//
// Which rows a workgroup has is worked out on the device: sequences' lengths are there, and a launch has as many blocks of rows as there may be at most.
#include "attention_core.h"

using namespace svdq;
using namespace svdq::attention;

namespace {

struct Params {
    const char *q, *k, *v;
    char *out;
    const int *cu_q, *cu_k, *lengths;
    float *partial;                        // keys in parts: [item][key head][row of the block] x D, then {maximum, sum} pairs
    long long qs[3], ks[3], vs[3], os[3];  // bytes: batch, token, head
    int S, Hkv, G, D, Tq, Tk, causal, zero_rest;
    int items, blocks;                     // per key head, at most
    int mirror;                            // rows form: the second so many items in the opposite order, see plan_of
    int target, least;                     // keys in parts (target > 0): about how many items in all, steps of one at least
    float scale2;                          // scale * log2(e)
};

__device__ inline int clamped(int x, int lo, int hi) { return x < lo ? lo : x < hi ? x : hi; }

// Rows of q that belong together: those of a sequence (s in 0 .. S - 1), or, packed, those in front of the first (region 0) and behind the last, which are in none.
// A launch has as many blocks as regions need that lie one behind the other, and nobody but its own region's workgroups may store a row: an offset below one in front of it
// counts as that one.  Offsets that are not in order so give fewer rows (and keys), never others, and every row is in one region.
struct Region {
    int s, first, count;  // sequence, its first query's row of q (of its batch entry, if they are not packed), its queries
    int key, keys;        // the same of k and v
};
__device__ inline int regions(const Params &p) { return p.cu_q ? p.S + 2 : p.S; }
__device__ inline int region_start(const Params &p, int i) { return i == 0 ? 0 : i > p.S + 1 ? p.Tq : clamped(p.cu_q[i - 1], 0, p.Tq); }  // (packed)
__device__ inline Region region_of(const Params &p, int i) {  // (packed: by its offsets as they stand)
    Region r;
    r.s = p.cu_q ? i - 1 : i;
    r.first = r.key = r.keys = 0;
    r.count = p.Tq;
    if (p.cu_q) {
        r.first = region_start(p, i);
        r.count = region_start(p, i + 1) - r.first;
    }
    if (r.s >= 0 && r.s < p.S) {
        if (p.cu_k) {
            r.key = clamped(p.cu_k[r.s], 0, p.Tk);
            r.keys = clamped(p.cu_k[r.s + 1], r.key, p.Tk) - r.key;
        } else {
            r.keys = p.lengths ? clamped(p.lengths[r.s], 0, p.Tk) : p.Tk;
        }
    }
    return r;
}
__device__ inline Region in_lane(const Region &r, int l) {
    return Region{__builtin_amdgcn_readlane(r.s, l), __builtin_amdgcn_readlane(r.first, l), __builtin_amdgcn_readlane(r.count, l), __builtin_amdgcn_readlane(r.key, l),
                  __builtin_amdgcn_readlane(r.keys, l)};
}
template <int ROWS>
__device__ inline int blocks_of(const Params &p, int count) {
    return (int)(((long long)count * p.G + ROWS - 1) / ROWS);
}

// op over this lane and those in front of it, by moves between lanes: 1, 2, 4 and 8 further in each 16, then the last of 16 and of 32 to those behind
template <typename F>
__device__ inline int up_to_lane(int x, F op) {  // (zero changes nothing)
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));
    return op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));
}
// (blocks are fewer than 2^24, parts 64 of each at most)
__device__ inline int sum_up_to_lane(int x) {
    return up_to_lane(x, [](int a, int b) __attribute__((always_inline)) { return a + b; });
}
__device__ inline int most_up_to_lane(int x) {
    return up_to_lane(x, [](int a, int b) __attribute__((always_inline)) { return a > b ? a : b; });
}
__device__ inline int most_of(int x) { return __builtin_amdgcn_readlane(most_up_to_lane(x), 63); }
__device__ inline float sum_of(float x) {
    return bits_f32(__builtin_amdgcn_readlane(
        up_to_lane((int)f32_bits(x), [](int a, int b) __attribute__((always_inline)) { return (int)f32_bits(bits_f32((uint32_t)a) + bits_f32((uint32_t)b)); }), 63));
}

// Packed, a region to a lane, in the order of the lanes: the one in front of them all begins at `before`
__device__ inline void put_in_order(const Params &p, Region &r, int before) {
    const int end = r.first + r.count, most = most_up_to_lane(r.first);
    r.first = most > before ? most : before;
    r.count = end > r.first && (p.zero_rest || (r.s >= 0 && r.s < p.S)) ? end - r.first : 0;
}

// A block of rows of a region and a part of its keys
struct Item {
    Region r;
    int rb, part, parts;
    int index, next;  // which of the items' partial results is its own, and how much further that of the next part is
    bool any;
};

// Item `at`.  A region's last block comes first: with a causal mask it has the most keys.
// Packed, up to 64 regions: their blocks one behind the other, which takes the sums over the regions in front of each.  (The workgroups without a block are the last ones
// then: between the others they leave some compute units with two and some with none, 16 sequences of 256, 12 heads of 64 20.8 us against 11.5.)
// More: region i has the numbers from f(i) = floor(start(i) * G / ROWS) + i to f(i + 1), as many as it needs or one or two more, without sums.  Its own is the last
// region whose f is not behind `at`, found among 64 at a time; in order are put the starts that are looked at, between those found before, so that all workgroups see the same ones.
template <int ROWS>
__device__ inline Item item_of(const Params &p, int at, int lane) {
    Item it;
    it.part = 0;
    it.parts = 1;
    it.index = it.next = 0;
    if (!p.cu_q) {
        it.r = region_of(p, at % p.S);
        it.rb = blocks_of<ROWS>(p, p.Tq) - 1 - at / p.S;
        it.any = true;
        return it;
    }
    int lo = 0, n = regions(p);
    if (n <= 64) {
        Region r = Region{0, 0, 0, 0, 0};
        if (lane < n) r = region_of(p, lane);
        put_in_order(p, r, 0);
        const int blocks = blocks_of<ROWS>(p, r.count);
        const int upto = sum_up_to_lane(blocks);
        const uint64_t behind = __ballot(at < upto);
        const int l = behind ? __builtin_ctzll(behind) : 0;
        it.r = in_lane(r, l);
        it.rb = __builtin_amdgcn_readlane(upto, l) - 1 - at;
        it.any = behind && it.rb < __builtin_amdgcn_readlane(blocks, l);
        return it;
    }
    int low = 0, high = p.Tq;  // where region `lo` begins and the last of the n ends
    for (;;) {
        const int step = (n + 63) / 64, i = lo + lane * step;
        Region r = Region{0, 0, 0, 0, 0};
        bool in = i < lo + n;
        int start = high;
        if (in) {
            if (step == 1) r = region_of(p, i);
            else r.first = region_start(p, i);
            start = clamped(r.first, low, high);
        }
        start = most_up_to_lane(start);
        in = in && (int)((long long)start * p.G / ROWS) + i <= at;
        const int l = 63 - __builtin_clzll(__ballot(in));  // (region `lo` itself is)
        low = __builtin_amdgcn_readlane(start, l);
        high = l < 63 ? __builtin_amdgcn_readlane(start, l + 1) : high;
        if (step == 1) {
            it.r = in_lane(r, l);
            it.r.first = low;
            it.r.count = p.zero_rest || (it.r.s >= 0 && it.r.s < p.S) ? high - low : 0;
            const int blocks = blocks_of<ROWS>(p, it.r.count), rel = at - ((int)((long long)low * p.G / ROWS) + lo + l);
            it.rb = blocks - 1 - rel;
            it.any = rel < blocks;
            return it;
        }
        lo += l * step;
        n = n - l * step < step ? n - l * step : step;
    }
}

// Item `at` where keys are divided into parts, or (BLOCK) the first of block `at`.  All regions' work together, in steps of SIZE keys, is divided by the number of items that
// is aimed at: longer keys than that are divided, evenly.  C regions to a lane.
constexpr int MAX_PARTS = 64, MAX_REGIONS = 256;
template <int ROWS, int SIZE, bool BLOCK, int C>
__device__ inline Item part_among(const Params &p, int at, int lane) {
    Region r[C];
    int blocks[C], steps[C], most = 0;
    float work = 0.f;
    const int n = regions(p);
#pragma unroll
    for (int c = 0; c < C; c++) {
        r[c] = Region{0, 0, 0, 0, 0};
        if (c * 64 + lane < n) r[c] = region_of(p, c * 64 + lane);
    }
    int before = 0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (p.cu_q) {
            put_in_order(p, r[c], before);
            before = __builtin_amdgcn_readlane(r[c].first, 63);
        }
        blocks[c] = blocks_of<ROWS>(p, r[c].count);
        steps[c] = (r[c].keys + SIZE - 1) / SIZE;
        if (blocks[c]) most = steps[c] > most ? steps[c] : most;
        work += (float)blocks[c] * (float)steps[c];
    }
    most = most_of(most);
    work = sum_of(work);
    int chunk = (int)__builtin_fminf(work / (float)p.target, 1.0e9f) + 1;
    chunk = chunk < p.least ? p.least : chunk;
    chunk = chunk < (most + MAX_PARTS - 1) / MAX_PARTS ? (most + MAX_PARTS - 1) / MAX_PARTS : chunk;
    Item it;
    it.any = false;
    int left = at, items_before = 0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (c * 64 >= n || it.any) continue;
        const int parts = steps[c] > chunk ? (steps[c] + chunk - 1) / chunk : 1;
        const int mine = blocks[c] * parts, items = sum_up_to_lane(mine), upto = BLOCK ? sum_up_to_lane(blocks[c]) : 0;  // of this region and those in front of it
        const uint64_t behind = __ballot(left < (BLOCK ? upto : items));
        if (behind) {
            const int l = __builtin_ctzll(behind), b = __builtin_amdgcn_readlane(blocks[c], l), before = __builtin_amdgcn_readlane(items, l) - __builtin_amdgcn_readlane(mine, l);
            it.r = in_lane(r[c], l);
            it.parts = __builtin_amdgcn_readlane(parts, l);
            const int rel = left - (BLOCK ? __builtin_amdgcn_readlane(upto, l) - b : before);  // (blocks of a part next to each other: they read the same keys)
            it.any = rel >= 0 && b > 0 && rel < b * (BLOCK ? 1 : it.parts);
            it.part = it.any ? rel / b : 0;
            it.rb = b - 1 - (rel - it.part * b);
            it.index = BLOCK ? items_before + before + rel : at;
            it.next = b;
        } else {
            left -= __builtin_amdgcn_readlane(BLOCK ? upto : items, 63);
            items_before += __builtin_amdgcn_readlane(items, 63);
        }
    }
    return it;
}

template <int ROWS, int SIZE, bool BLOCK>
__device__ inline Item part_of(const Params &p, int at, int lane) {
    return regions(p) <= 64 ? part_among<ROWS, SIZE, BLOCK, 1>(p, at, lane) : part_among<ROWS, SIZE, BLOCK, MAX_REGIONS / 64>(p, at, lane);
}

// This lane's row, and the keys that rows see
struct Rows {
    const char *q;
    char *out;
    int total, off, keys, limit;  // rows of the sequence; key of its first query; keys; the row sees the keys in front of `limit`
    bool in;
};
__device__ inline int limit_of(const Params &p, const Rows &r, int row) { return p.causal ? clamped(row / p.G + r.off + 1, 0, r.keys) : r.keys; }
__device__ inline Rows rows_of(const Params &p, const Region &g, int hk, int row) {
    Rows r;
    const int t = row / p.G, head = hk * p.G + (row - t * p.G);
    const long long entry = p.cu_q ? 0 : g.s;
    r.total = g.count * p.G;
    r.off = g.keys - g.count;
    r.keys = g.keys;
    r.in = row < r.total;
    r.q = p.q + entry * p.qs[0] + (long long)(g.first + t) * p.qs[1] + head * p.qs[2];
    r.out = p.out + entry * p.os[0] + (long long)(g.first + t) * p.os[1] + head * p.os[2];
    r.limit = limit_of(p, r, row);
    return r;
}
// The limits of the first of `count` rows from `row` on and of the last one of the sequence among them (none: zero keys)
__device__ inline void limits_of(const Params &p, const Rows &r, int row, int count, int &least, int &most) {
    const int last = row + count < r.total ? row + count - 1 : r.total - 1;
    least = limit_of(p, r, row);
    most = last < row ? 0 : limit_of(p, r, last);
}
__device__ inline const char *first_key(const Params &p, const Region &g, const char *t, const long long (&s)[3], int hk) {
    return t + (p.cu_k || g.s < 0 || g.s >= p.S ? 0 : g.s) * s[0] + g.key * s[1] + hk * s[2];
}

template <bool BF16, typename H>
__device__ inline void load_q(const Params &p, typename Elem<BF16>::vec (&qf)[H::KS], const Rows &r, int lane) {
#pragma unroll
    for (int ks = 0; ks < H::KS; ks++) {
        const int c = 16 * ks + 8 * (lane >> 5);
        u32x4_t w = u32x4_t{0, 0, 0, 0};
        if (r.in && c < p.D) w = *(const u32x4_t *)(r.q + c * 2);
        qf[ks] = __builtin_bit_cast(typename Elem<BF16>::vec, w);
    }
}
template <bool BF16, typename H>
__device__ inline void wait_for_q(typename Elem<BF16>::vec (&qf)[H::KS]) {
#pragma unroll
    for (int ks = 0; ks < H::KS; ks++) asm volatile("" : "+v"(qf[ks]));
}

// The first step of a part, of those that all of the sequence's keys make
template <int SIZE>
__device__ inline int first_step(const Item &it, int part) {
    const int all = (it.r.keys + SIZE - 1) / SIZE, each = all / it.parts, more = all - each * it.parts;
    return part * each + (part < more ? part : more);
}
// The steps of an item, no more than those of the first `most` keys, which its block sees.  With a causal mask parts may lie behind those: nobody has to do anything for them
// (false), and a block whose keys end in its first part is whole.
template <int SIZE>
__device__ inline bool share(Item &it, int most, int &begin, int &end) {
    begin = 0;
    end = (most + SIZE - 1) / SIZE;
    if (it.parts == 1) return true;
    begin = first_step<SIZE>(it, it.part);
    const int stop = first_step<SIZE>(it, it.part + 1);
    if (it.part == 0 && stop >= end) it.parts = 1;
    if (it.part > 0 && begin >= end) return false;
    end = stop < end ? stop : end;
    return true;
}
// Where an item's share of a row goes, and its maximum and sum behind all of those
template <int ROWS>
__device__ inline float *share_of(const Params &p, int index, int hk, int row) {
    return p.partial + (((long long)index * p.Hkv + hk) * ROWS + row) * p.D;
}
template <int ROWS>
__device__ inline float *stats_of(const Params &p, int index, int hk, int row) {
    return p.partial + (long long)p.items * p.Hkv * ROWS * p.D + (((long long)index * p.Hkv + hk) * ROWS + row) * 2;
}

// A step in which some rows do not see some keys, where what such a key has in V is an infinity or a NaN: zero times it is a NaN, too.  A key at a time; rows that
// do not see it keep what they have.
template <bool BF16, typename H, int NB, typename S, typename F>
__device__ inline void attend_key_by_key(S &st, const float16_t (&s)[NB], const char *v, int first, int limit, int lane, F &&probabilities) {
    using vec = typename Elem<BF16>::vec;
#pragma unroll
    for (int n = 0; n < 2 * NB; n++) {
        vec vf[H::DB];
        st.read_v(vf, v, n, lane);
        const u32x4_t pr = __builtin_bit_cast(u32x4_t, probabilities(n));
#pragma unroll 1
        for (int j = 0; j < 16; j++) {  // (element 4 (j / 8) + j % 4 of the half-wave j / 4 % 2)
            const int at = 4 * (j >> 3) + (j & 3);
            const bool half = (lane >> 5) == ((j >> 2) & 1), seen = first + 16 * n + j < limit;
            u32x4_t keep;
#pragma unroll
            for (int w = 0; w < 4; w++) keep[w] = half && at >> 1 == w ? (at & 1 ? 0xFFFF0000u : 0xFFFFu) : 0u;
            const vec p = __builtin_bit_cast(vec, pr & keep);
#pragma unroll
            for (int d = 0; d < H::DB; d++) {
                const float16_t o = Elem<BF16>::mfma(__builtin_bit_cast(vec, __builtin_bit_cast(u32x4_t, vf[d]) & keep), p, st.o[d]);
#pragma unroll
                for (int e = 0; e < 16; e++) st.o[d][e] = seen ? o[e] : st.o[d][e];
            }
        }
    }
}
// whether a sum of this wave's is a NaN or an infinity, of the head's columns (what stands behind them in LDS is nobody's)
template <bool BF16, typename H>
__device__ inline bool any_nan(const State<BF16, H> &st, int D) {
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < H::DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (32 * d + 8 * (e >> 2) < D) x = __builtin_fmaf(st.o[d][e], 0.f, x);
    return __any(x != x);
}

// keys that a row does not see get a score of minus infinity: those from `limit` on, of NB blocks of 32 from key `first` on
template <int NB>
__device__ inline void hide(float16_t (&s)[NB], int first, int limit, int lane) {
    const int left = limit - first - 4 * (lane >> 5);
#pragma unroll
    for (int kb = 0; kb < NB; kb++)
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (32 * kb + 8 * (e >> 2) + (e & 3) >= left) s[kb][e] = -__builtin_huge_valf();
}

// ---- keys form: 32 rows per workgroup, whose waves take every fourth step (of 32 keys) of the part's keys, each through its own LDS, a
// step ahead, and meet in LDS at the end; the parts of a row block meet in self_attention_join_kernel ------------------------------------
template <bool BF16, int DP>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1) self_attention_keys_kernel(Params p) {
    using H = Head<DP, true>;
    using E = Elem<BF16>;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv, at = blockIdx.x / p.Hkv;
    constexpr int SIZE = 32;
    Item it = p.target ? part_of<32, SIZE, false>(p, at, lane) : item_of<32>(p, at, lane);
    if (!it.any) return;
    const Rows r = rows_of(p, it.r, hk, it.rb * 32 + col);
    int least, most, begin, end;
    limits_of(p, r, it.rb * 32, 32, least, most);
    if (!share<SIZE>(it, most, begin, end)) return;
    typename E::vec qf[H::KS];
    load_q<BF16, H>(p, qf, r, lane);
    const char *kp = first_key(p, it.r, p.k, p.ks, hk), *vp = first_key(p, it.r, p.v, p.vs, hk);
    constexpr int REQ = H::REQ / 2, STAGE = H::TILE;  // a stage: 32 rows of K, then of V
    char *mine = lds + wave * 2 * STAGE;
    const uint32_t area = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + wave * 2 * STAGE;
    const int bytes = p.D * 2;
    // Request i brings rows r0 + i * RPR: of V the same piece every time, of K the pieces that f has there
    const int r0 = lane / H::PIECES, ck = ((lane % H::PIECES) ^ H::fk(r0)) * 16, cv = ((lane % H::PIECES) ^ H::fv(r0)) * 16;
    const uint32_t ok = (uint32_t)(r0 * p.ks[1]), ov = (uint32_t)(r0 * p.vs[1]) + cv;
    static_assert(H::fv(H::RPR) == 0 && (H::RPR == 16 || H::fk(H::RPR) == 4), "");
    // columns behind the head's end are zero in K for good (the wait for a step's copies is one for these, too)
    zero_columns<H, SIZE>(mine, p.D / 8, lane, 64);
    zero_columns<H, SIZE>(mine + STAGE, p.D / 8, lane, 64);
    auto request = [&](int step, int slot) __attribute__((always_inline)) {
        const char *k = kp + (long long)step * SIZE * p.ks[1], *v = vp + (long long)step * SIZE * p.vs[1];
        const int left = most - step * SIZE;
        const uint32_t dst = area + slot * STAGE;
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            const int c = ck ^ (64 * (i & (16 / H::RPR - 1)));
            if (c < bytes && r0 < left - i * H::RPR) copy16(dst + i * 1024, k + i * H::RPR * p.ks[1], ok + c);
        }
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            if (cv >= bytes) continue;
            if (r0 < left - i * H::RPR) copy16(dst + STAGE / 2 + i * 1024, v + i * H::RPR * p.vs[1], ov);
            else clear16(dst + STAGE / 2 + i * 1024 + lane * 16);
        }
    };
    State<BF16, H> st;
    // Once more, key by key where rows do not see all keys, if sums turn out to hold a NaN: rows that see none of its causes have none then
    for (bool careful = false;; careful = true) {
        st.clear();
        int step = begin + wave;
        if (step < end) request(step, 0);
        wait_for_q<BF16, H>(qf);
        for (int slot = 0; step < end; slot ^= 1) {
            const int next = step + 4;
            if (next < end) request(next, slot ^ 1);
            // This step's copies have landed when no more than the next one's are on their way.  Of a step with keys behind the last one some
            // requests may have had no lane to make them: then all have to land.
            if (next < end && most - next * SIZE >= SIZE) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * REQ) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            const char *k = mine + slot * STAGE + col * H::PITCH, *v = mine + slot * STAGE + STAGE / 2;
            float16_t s[1];
#pragma unroll
            for (int e = 0; e < 16; e++) s[0][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < H::KS; ks++) {
                const u32x4_t w = *(const u32x4_t *)(k + ((2 * ks + h) ^ H::fk(col)) * 16);
                s[0] = E::mfma(__builtin_bit_cast(typename E::vec, w), qf[ks], s[0]);
            }
            const bool some = least < (step + 1) * SIZE;
            if (some) hide(s, step * SIZE, r.limit, lane);
            if (some && careful) {
                st.raise(st.highest(s), p.scale2);
                const float ref = st.reference();
                attend_key_by_key<BF16, H>(st, s, v, step * SIZE, r.limit, lane, [&](int n) __attribute__((always_inline)) { return st.template exponentials<1, false>(s, n, p.scale2, ref); });
            }
            else st.template attend<false>(s, 0xFFFFFFFFull, p.scale2, v, lane);
            step = next;
        }
        if (careful || !p.causal || !any_nan(st, p.D)) break;
    }
    // The waves meet.  Each leaves its maximum, sum and outputs in the place of its own stages, 16 columns (a unit) of 64 lanes in 2 KB, and takes
    // every fourth unit of all four, scaled to the highest maximum.
    constexpr int UNITS = 2 * H::DB, AREA = 2 * STAGE;
    static_assert(256 + UNITS * 2048 <= AREA, "");
    const float own = across_sum(st.sum);
    if (h == 0) {
        ((float *)mine)[col] = st.top;
        ((float *)mine)[32 + col] = own;
    }
    if (r.in) {
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
    const float inv = inverse(sum);
    float *dst = share_of<32>(p, it.index, hk, col);
    const int columns = r.in ? p.D : 0;
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
            if (it.parts > 1 && c < columns) *(float4_t *)(dst + c) = y;
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * i + e] = y[e];
        }
        if (it.parts == 1) store_columns<BF16>(r.out, x, inv, 16 * u, columns, lane);
    }
    if (it.parts > 1 && wave == 0 && h == 0 && r.in) {
        float *ms = stats_of<32>(p, it.index, hk, col);
        ms[0] = top;
        ms[1] = sum;
    }
}

// ---- the running softmax of 32 rows, as the forms below have it that are bound by their vector instructions ----------------------------
// The sums of the (rounded) probabilities come from the matrix cores, too: v_mfma_f32_16x16x32 takes the same registers for sixteen rows' 32 keys, of which lanes 16 .. 31 and 48 .. 63
// hold those of sixteen other rows; a left operand whose row 0 has ones for the first and third eight keys, and row 1 for the others, adds both apart.  16 cycles
// of the matrix cores for 8 additions of 4 cycles, and both sides of the division have the same roundings.  (A NaN of one of two such rows is a NaN in both their sums, since
// nothing times it is one: then the wave's rows are worked out once more, with sums of their own.)
template <bool BF16>
__device__ inline float4_t add_up(typename Elem<BF16>::vec ones, typename Elem<BF16>::vec p, float4_t c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p, c, 0, 0, 0);
}
template <bool BF16, typename H>
struct Softmax : State<BF16, H> {
    using E = Elem<BF16>;
    using vec = typename E::vec;
    using Base = State<BF16, H>;
    float4_t sums;  // lanes 0 .. 15: of rows 0 .. 15 and 16 .. 31
    vec ones;
    __device__ inline void start(int lane) {
        const uint32_t w = (lane & 15) == ((lane >> 4) & 1) ? E::ONE * 0x10001u : 0u;
        ones = __builtin_bit_cast(vec, u32x4_t{w, w, w, w});
    }
    __device__ inline void clear() {
        Base::clear();
        sums = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    // (a maximum that a NaN stays in takes no instructions of its own to make quiet ones of others)
    static __device__ inline float highest(const float16_t (&s)[2]) {
        float m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            m[i] = s[i >> 1][8 * (i & 1)];
#pragma unroll
            for (int e = 1; e < 8; e++) m[i] = __builtin_elementwise_maximum(m[i], s[i >> 1][8 * (i & 1) + e]);
        }
        return across_max(__builtin_elementwise_maximum(__builtin_elementwise_maximum(m[0], m[1]), __builtin_elementwise_maximum(m[2], m[3])));
    }
    // Whether a step's maximum has to be looked for.  In bf16, every LOOKS-th alone: probabilities have fp32's range, and sums of 2^64 or more, or an infinity or a NaN among the
    // outputs, send the rows through `attend_carefully`, which looks at every step.  As long as a row has no reference at all, at every step, so that its sums are zero when it gets
    // one.  (In fp16 a rise of 2^9 between two looks would be beyond the range.)  16384 tokens, 8 heads of 128 897 -> 863 us, 8192 tokens, 16 heads of 64
    // 299 -> 284, 4608 tokens, 24 heads of 72 189 -> 180, 1024 tokens, 24 heads of 128 23.8 -> 23.4.  The price: finite scores that rise by 44 or more between two looks are
    // worked out twice, the second time without overlap.  The same three, one key 90 above those in front of it: 860 -> 1980, 283 -> 651, 178 -> 425.
    static constexpr int LOOKS = 8;
    __device__ inline bool due(int step) const { return !BF16 || step % LOOKS == 0 || __any(this->top == -__builtin_huge_valf()); }
    __device__ inline void raise(float high, float scale2, int lane) {
        if (__any(__builtin_fmaf(high, scale2, -this->top) > E::RAISED + 8.f)) {
            const float m = high * scale2 - E::RAISED, now = m > this->top ? m : this->top;
            const float f = this->top == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(this->top - now);
            this->top = now;
#pragma unroll
            for (int d = 0; d < H::DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) this->o[d][e] *= f;
            if (!H::ONES) {
                sums[0] *= f;
                sums[1] *= __shfl(f, (lane & 15) + 16);
            }
        }
    }
    // the right operand: probabilities of 16 keys, rounded
    __device__ inline vec exponentials(const float16_t (&s)[2], int n, float scale2, float ref) { return Base::template exponentials<2, true>(s, n, scale2, ref); }
    __device__ inline void add(vec p) {
        if (!H::ONES) sums = add_up<BF16>(ones, p, sums);
    }
    // A step's scores and values (v in LDS) join the sums, 16 keys at a time: while the matrix cores multiply the probabilities of one 16, those of the next are made and
    // the operands of the one behind it are on their way.
    __device__ inline void attend(const float16_t (&s)[2], float scale2, bool look, const char *v, int lane) {
        vec vf[2][H::DB], pr[2];
        Base::read_v(vf[0], v, 0, lane);
        if (look) raise(highest(s), scale2, lane);
        const float ref = this->reference();
        pr[0] = exponentials(s, 0, scale2, ref);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 4; n++) {
            if (n < 3) {
                Base::read_v(vf[(n + 1) & 1], v, n + 1, lane);
                pr[(n + 1) & 1] = exponentials(s, n + 1, scale2, ref);
            }
#pragma unroll
            for (int d = 0; d < H::DB; d++) this->o[d] = E::mfma(vf[n & 1][d], pr[n & 1], this->o[d]);
            add(pr[n & 1]);
            if (n < 3) {
#pragma unroll
                for (int d = 0; d < H::DB; d++) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 16 / H::DB, 0);
                    __builtin_amdgcn_sched_group_barrier(0x400, 8 / H::DB, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the same with sums by additions, and, where some rows do not see all keys, key by key
    __device__ inline void attend_carefully(float16_t (&s)[2], float scale2, const char *v, int first, int limit, bool some, int lane) {
        if (!some) {
            Base::template attend<H::ONES>(s, ~0ull, scale2, v, lane);
            return;
        }
        Base::raise(Base::highest(s), scale2);
        const float ref = this->reference();
        attend_key_by_key<BF16, H>(*this, s, v, first, limit, lane, [&](int n) __attribute__((always_inline)) { return Base::template exponentials<2, H::ONES>(s, n, scale2, ref); });
    }
    // whether what there is may hold a NaN that belongs to another row, or to a key that a row does not see, or comes from an old maximum
    __device__ inline bool doubtful(bool causal, int D, int lane) const {
        float x = H::ONES || lane >= 16 ? 0.f : __builtin_fmaxf(sums[0], sums[1]) + (sums[0] + sums[1]) * 0.f;
        if constexpr (BF16 && H::ONES) x = whole_sum(D, false, lane);
        return __any(!(x < 0x1p64f)) || ((BF16 || causal) && any_nan(*(const Base *)this, D));
    }
    // of this lane's row
    __device__ inline float whole_sum(int D, bool careful, int lane) const {
        if constexpr (H::ONES) {
            float x = 0.f;
#pragma unroll
            for (int g = 0; g < 4 * H::DB; g++)
                if (8 * g == D && lane < 32) x = this->o[g >> 2][4 * (g & 3)];
            return across_sum(x);
        }
        if (careful) return across_sum(this->sum);
        const float low = __shfl(sums[0], lane & 15), high = __shfl(sums[1], lane & 15);
        return lane & 16 ? high : low;
    }
};

// The end of a wave's 32 rows: the quotients
template <bool BF16, typename H>
__device__ inline void finish(const Params &p, const Rows &r, const Softmax<BF16, H> &st, bool careful, int lane) {
    const float inv = inverse(st.whole_sum(p.D, careful, lane));
#pragma unroll
    for (int u = 0; u < 2 * H::DB; u++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = st.o[u >> 1][8 * (u & 1) + e];
        store_columns<BF16>(r.out, x, inv, 16 * u, r.in ? p.D : 0, lane);
    }
}
// or an item's share of them
template <bool BF16, typename H, int BLOCK_ROWS>
__device__ inline void finish_part(const Params &p, const Item &it, const Rows &r, const Softmax<BF16, H> &st, bool careful, int hk, int wave, int lane) {
    const int col = lane & 31, h = lane >> 5;
    const float sum = st.whole_sum(p.D, careful, lane);
    if (!r.in) return;
    float *dst = share_of<BLOCK_ROWS>(p, it.index, hk, wave * 32 + col);
#pragma unroll
    for (int d = 0; d < H::DB; d++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int c = 32 * d + 8 * g + 4 * h;
            if (c < p.D) *(float4_t *)(dst + c) = float4_t{st.o[d][4 * g], st.o[d][4 * g + 1], st.o[d][4 * g + 2], st.o[d][4 * g + 3]};
        }
    if (h == 0) {
        float *ms = stats_of<BLOCK_ROWS>(p, it.index, hk, wave * 32 + col);
        ms[0] = st.top;
        ms[1] = sum;
    }
}

// ---- rows form: 128 rows per workgroup, 32 per wave; all four waves share the keys through LDS, 64 a step, two steps of them; two workgroups or three to a compute
// unit.  Where rows are fewer than whole blocks of the turns form would have for every compute unit ---------------------------------------------------------------
constexpr int HALF = 128;

template <bool BF16, int DP, bool ONES>
__global__ void __launch_bounds__(256, DP <= 32 ? 4 : DP <= 64 ? 3 : 2) self_attention_rows_kernel(Params p) {
    using H = Head<DP, false, ONES>;
    using E = Elem<BF16>;
    using vec = typename E::vec;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv;
    int at = blockIdx.x / p.Hkv;
    if (at >= p.mirror && at < 2 * p.mirror) at = p.mirror + (2 * p.mirror < p.items ? 2 * p.mirror : p.items) - 1 - at;
    Item it = p.target ? part_of<HALF, KEYS, false>(p, at, lane) : item_of<HALF>(p, at, lane);
    if (!it.any) return;
    const int wave0 = it.rb * HALF + wave * 32;
    Rows r = rows_of(p, it.r, hk, wave0 + col);
    int least, most, wave_least, wave_most, begin, end;
    limits_of(p, r, it.rb * HALF, HALF, least, most);
    limits_of(p, r, wave0, 32, wave_least, wave_most);
    vec qf[H::KS];
    load_q<BF16, H>(p, qf, r, lane);
    // a part's keys: limits from its first one on
    if (!share<KEYS>(it, most, begin, end)) return;
    const int skip = begin * KEYS, stop = end * KEYS;
    most = (most < stop ? most : stop) - skip;
    wave_most = (wave_most < stop ? wave_most : stop) - skip;
    wave_least -= skip;
    r.limit -= skip;
    const int steps = end > begin ? end - begin : 0;
    Copies<H, 4> copies(lds, first_key(p, it.r, p.k, p.ks, hk) + skip * p.ks[1], first_key(p, it.r, p.v, p.vs, hk) + skip * p.vs[1], p.ks[1], p.vs[1], p.D, most, wave, lane, E::ONE);
    Softmax<BF16, H> st;
    st.start(lane);
    auto ask = [&](int step, int slot) __attribute__((always_inline)) {
        const int left = most - step * KEYS;
        copies.k(step, slot);
        copies.v(step, slot, left >= KEYS ? ~0ull : (1ull << left) - 1);
    };
    float16_t s[2];
    // operands of four matrix instructions at a time, the next four's on their way
    constexpr int N = 2 * H::KS, GROUP = N % 4 == 0 ? 4 : 2;
    auto score = [&](int slot) __attribute__((always_inline)) {
        const char *k = lds + slot * H::TILE + col * H::PITCH;
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
    };
    st.clear();
    if (steps > 0) ask(0, 0);
    wait_for_q<BF16, H>(qf);
    for (int step = 0; step < steps; step++) {
        const int slot = step & 1;
        // K and V of this step have landed, of all waves, and nobody reads what the next requests overwrite
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + 1 < steps) ask(step + 1, slot ^ 1);
        if (step * KEYS >= wave_most) continue;
        if (DP > 64) __builtin_amdgcn_s_setprio(1);  // (8 heads of 128, 16384 tokens 1001 -> 984 us; heads of 64 301 -> 303)
        score(slot);
        if (DP > 64) __builtin_amdgcn_s_setprio(0);
        if (wave_least < (step + 1) * KEYS) hide(s, step * KEYS, r.limit, lane);
        st.attend(s, p.scale2, st.due(step), lds + (2 + slot) * H::TILE, lane);
    }
    // Once more, and key by key where rows do not see all keys, if there turns out to be a NaN: rows that see none of its causes have none then
    bool careful = false;
    if (steps > 0) {
        int *flags = (int *)(lds + 4 * H::TILE);
        const bool nan = st.doubtful(p.causal, p.D, lane);
        if (lane == 0) flags[wave] = nan;
        __syncthreads();
        careful = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]) != 0;
        if (careful) {
            st.clear();
#pragma unroll 1
            for (int step = 0; step < steps; step++) {
                asm volatile("s_barrier" ::: "memory");
                ask(step, 0);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (step * KEYS >= wave_most) continue;
                score(0);
                const bool some = wave_least < (step + 1) * KEYS;
                if (some) hide(s, step * KEYS, r.limit, lane);
                st.attend_carefully(s, p.scale2, lds + 2 * H::TILE, step * KEYS, r.limit, some, lane);
            }
        }
    }
    if (it.parts > 1) finish_part<BF16, H, HALF>(p, it, r, st, careful, hk, wave, lane);
    else finish<BF16, H>(p, r, st, careful, lane);
}

// ---- turns form: 256 rows per workgroup, 32 per wave; all eight waves share the keys through LDS, 64 a step, four steps of them -----------
// The two waves of a SIMD take turns: while one makes probabilities of its scores (vector instructions), the other multiplies (the probabilities before
// those with V, the next keys with Q).  A phase is one or the other; waves 4 .. 7 are one phase behind waves 0 .. 3, and a barrier ends a phase for all.
// In phase 2 j the first four waves make the probabilities of step j, in phase 2 j + 1 they multiply them and score step j + 1.  Keys and values of step i are
// read in phases 2 i - 1 .. 2 i + 2; those of step i + 4 take their place.  Every wave asks for its share of them where it makes probabilities, in phases 2 i + 3 and 2 i + 4, and
// waits for it at the end of phase 2 i + 6 (asking between the matrix instructions: 8 heads of 128, 16384 tokens 953 -> 922 us).
constexpr int STAGES = 4, WAVES = 8, ROWS = 32 * WAVES;

__device__ inline void phase_ends() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A wave's share of the copies: the same requests at every step, of K by the first four waves, of V by the others
template <typename H>
struct RowCopies {
    static constexpr int REQ = 2 * H::REQ / WAVES;
    static_assert(REQ * WAVES == 2 * H::REQ && H::REQ % REQ == 0, "");
    const char *first, *next;  // of the first step, of the one to be asked for next
    long long bytes;           // a step
    uint32_t dst, off[REQ];
    uint64_t in[REQ];  // lanes whose piece lies in the head
    int row[REQ], most, steps, whole;
    bool values;
    __device__ inline RowCopies(const Params &p, char *lds, const char *kp, const char *vp, int most_, int wave, int lane) {
        values = wave >= WAVES / 2;
        first = next = values ? vp : kp;
        const long long token = values ? p.vs[1] : p.ks[1];
        bytes = KEYS * token;
        most = most_;
        whole = most > 0 ? most / KEYS : 0;
        steps = most > 0 ? (most + KEYS - 1) / KEYS : 0;
        const int request = (wave - (values ? WAVES / 2 : 0)) * REQ;
        dst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (values ? STAGES * H::TILE : 0) + request * 1024;
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            const int piece = (request + i) * 64 + lane, place = piece % H::PIECES;
            row[i] = piece / H::PIECES;
            const int c = (place ^ (values ? H::fv(row[i]) : H::fk(row[i]))) * 16;
            off[i] = (uint32_t)(row[i] * token) + c;
            in[i] = __ballot(c < p.D * 2);
        }
    }
    // Rows behind the last key are not read: their scores are masked whatever K holds, and V holds zeros there, since nothing times a NaN is one.
    __device__ inline void ask_at(const char *src, int step, int slot) const {
        const uint32_t to = dst + slot * H::TILE;
        const int left = most - step * KEYS, lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < REQ; i++) {
            if (!(in[i] >> lane & 1)) continue;
            if (row[i] < left) copy16(to + i * 1024, src, off[i]);
            else if (values) clear16(to + i * 1024 + lane * 16);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a barrier alone does not wait for LDS)
    }
    // The next step.  Of a whole one, all lanes of all requests, or (a head that ends inside a row of LDS) all requests in one piece, without branches around those lanes that
    // have none.  What a request costs is its issue, about 25 cycles of the compute unit whatever its lanes bring: rows of 192 bytes instead of 256 for heads of 72 .. 96 are
    // three requests a wave instead of four (4608 tokens, 24 heads of 72 199 -> 186 us, 8192 tokens, 16 heads of 96 383 -> 363).
    __device__ inline void ask(int step, int slot) {
        if (step < whole) {
            const uint32_t to = dst + slot * H::TILE;
            [[maybe_unused]] uint64_t lanes;
            if constexpr (!H::ONES) {
#pragma unroll
                for (int i = 0; i < REQ; i++) copy16(to + i * 1024, next, off[i]);
            } else if constexpr (REQ == 4) {
                asm volatile(
                    "s_mov_b64 %0, exec\n\t"
                    "s_mov_b32 m0, %1\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %7, %2\n\t"
                    "s_add_u32 m0, m0, 0x400\n\ts_mov_b64 exec, %4\n\tglobal_load_lds_dwordx4 %8, %2\n\t"
                    "s_add_u32 m0, m0, 0x400\n\ts_mov_b64 exec, %5\n\tglobal_load_lds_dwordx4 %9, %2\n\t"
                    "s_add_u32 m0, m0, 0x400\n\ts_mov_b64 exec, %6\n\tglobal_load_lds_dwordx4 %10, %2\n\t"
                    "s_mov_b64 exec, %0"
                    : "=&s"(lanes)
                    : "s"(to), "s"(next), "s"(in[0]), "s"(in[1]), "s"(in[2]), "s"(in[3]), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3])
                    : "memory", "m0", "scc");
            } else {
                static_assert(REQ == 3, "");
                asm volatile(
                    "s_mov_b64 %0, exec\n\t"
                    "s_mov_b32 m0, %1\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %6, %2\n\t"
                    "s_add_u32 m0, m0, 0x400\n\ts_mov_b64 exec, %4\n\tglobal_load_lds_dwordx4 %7, %2\n\t"
                    "s_add_u32 m0, m0, 0x400\n\ts_mov_b64 exec, %5\n\tglobal_load_lds_dwordx4 %8, %2\n\t"
                    "s_mov_b64 exec, %0"
                    : "=&s"(lanes)
                    : "s"(to), "s"(next), "s"(in[0]), "s"(in[1]), "s"(in[2]), "v"(off[0]), "v"(off[1]), "v"(off[2])
                    : "memory", "m0", "scc");
            }
        } else if (step < steps) {
            ask_at(next, step, slot);
        }
        next += bytes;
    }
    // Step j + 1 has landed.  Step j + 2 alone has been asked for behind it; of the last step some requests may have had no lane to make them.
    __device__ inline void wait_for_next(int j) const {
        if (j + 3 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(REQ) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};

template <bool BF16, int DP, bool ONES>
__global__ void __launch_bounds__(512, 2) self_attention_turns_kernel(Params p) {
    using H = Head<DP, false, ONES>;
    using E = Elem<BF16>;
    using vec = typename E::vec;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % p.Hkv, at = blockIdx.x / p.Hkv;
    const Item it = item_of<ROWS>(p, at, lane);
    if (!it.any) return;
    const int wave0 = it.rb * ROWS + wave * 32;
    const Rows r = rows_of(p, it.r, hk, wave0 + col);
    int least, most, wave_least, wave_most;
    limits_of(p, r, it.rb * ROWS, ROWS, least, most);
    limits_of(p, r, wave0, 32, wave_least, wave_most);
    vec qf[H::KS];
    load_q<BF16, H>(p, qf, r, lane);
    RowCopies<H> copies(p, lds, first_key(p, it.r, p.k, p.ks, hk), first_key(p, it.r, p.v, p.vs, hk), most, wave, lane);
    const int steps = copies.steps;
    const bool late = wave >= WAVES / 2;
    const int ahead = late ? STAGES - 1 : STAGES - 2;  // steps
    for (int i = 0; i < ahead; i++) copies.ask(i, i);
    // columns behind the head's end, as far as they are multiplied, are zero in K for good: no copy writes there
    zero_columns<H, STAGES * KEYS>(lds, p.D / 8, threadIdx.x, 64 * WAVES);
    if constexpr (H::ONES) {
        for (int i = threadIdx.x; i < STAGES * KEYS; i += 64 * WAVES)
            *(u32x4_t *)(lds + STAGES * H::TILE + i * H::PITCH + ((p.D / 8) ^ H::fv(i)) * 16) = u32x4_t{E::ONE, 0, 0, 0};
    }
    Softmax<BF16, H> st;
    st.start(lane);
    st.clear();
    float16_t s[2];
    // Operands of the matrix instructions of a phase: 0 .. VALUES - 1 sixteen keys' values of 32 columns, for their probabilities, then 32 keys of the next step.  Eight are there
    // or on their way; where one has been multiplied, that of the eighth instruction behind takes its place.
    constexpr int VALUES = 4 * H::DB, ALL = VALUES + 2 * H::KS, AHEAD = 8;
    static_assert(VALUES >= AHEAD, "");  // (keys have not landed where the first operands are asked for)
    vec pr[4], ops[AHEAD];
    // Where this lane's operands stand in LDS: with what differs between the instructions of a phase by an exclusive or, worked out anew each time (registers are short)
    typedef __attribute__((address_space(3))) char *lds_t;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t)lds;
    const uint32_t k_lane = lds0 + col * H::PITCH + (h ^ H::fk(col)) * 16;
    const uint32_t v_lane = lds0 + STAGES * H::TILE + (4 * h + ((lane & 15) >> 2)) * H::PITCH + (lane & 1) * 8 + ((((lane >> 4) & 1) * 2 + ((lane >> 1) & 1)) ^ H::fv((lane & 15) >> 2)) * 16;
    uint32_t k_at, v_at;  // of the next step's keys, of a step's values
    auto read = [&](int i) __attribute__((always_inline)) {
        if (i < VALUES) {
            typedef short short4_t __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4_t *tr_t;
            const lds_t at = (lds_t)(uintptr_t)((H::PITCH == 256 ? v_at ^ (i % H::DB * 64) : v_at + i % H::DB * 64) + i / H::DB * 16 * H::PITCH);
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)(at + 8 * H::PITCH));
            ops[i % AHEAD] = __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int n = i - VALUES, kb = n & 1, ks = n >> 1;
            ops[i % AHEAD] = __builtin_bit_cast(vec, *(__attribute__((address_space(3))) u32x4_t *)(uintptr_t)((H::PITCH == 256 ? k_at ^ (ks * 32) : (k_at ^ (ks % 2 * 32)) + ks / 2 * 64) + kb * 32 * H::PITCH));
        }
    };
    auto stand = [&](int slot) __attribute__((always_inline)) {
        v_at = v_lane + slot * H::TILE;
        k_at = k_lane + (slot + 1) % STAGES * H::TILE;
        asm volatile("" : "+v"(v_at), "+v"(k_at));
    };
    auto multiply = [&](auto from, auto to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = from; i < to; i++) {
            if (i == VALUES) {
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[kb][e] = 0.f;
            }
            if (i < VALUES) {
                st.o[i % H::DB] = E::mfma(ops[i % AHEAD], pr[i / H::DB], st.o[i % H::DB]);
                if (i % H::DB == H::DB - 1) st.add(pr[i / H::DB]);
            } else {
                const int n = i - VALUES, kb = n & 1, ks = n >> 1;
                s[kb] = E::mfma(ops[i % AHEAD], qf[ks], s[kb]);
            }
            if (i + AHEAD < ALL) read(i + AHEAD);  // (behind a row's last step, of keys that are not multiplied)
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> FIRST;
    constexpr std::integral_constant<int, VALUES> SCORES;
    constexpr std::integral_constant<int, ALL> END;
    // the scores of the step in `slot`, from nothing
    auto score = [&](int slot) __attribute__((always_inline)) {
        stand((slot + STAGES - 1) % STAGES);
#pragma unroll
        for (int i = 0; i < AHEAD && VALUES + i < ALL; i++) read(VALUES + i);
        multiply(SCORES, END);
    };
    bool careful = false;
    if (steps > 0) {
        wait_for_q<BF16, H>(qf);
        if (steps > STAGES - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(RowCopies<H>::REQ * (STAGES - 3)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        phase_ends();
        if (late) phase_ends();
        if (wave_most > 0) score(0);
        if (late) copies.wait_for_next(0);
        phase_ends();
        for (int j = 0; j < steps; j++) {
            const int slot = j % STAGES;
            const bool here = j * KEYS < wave_most;
            copies.ask(j + ahead, (j + ahead) % STAGES);
            if (here) {
                if (wave_least < (j + 1) * KEYS) hide(s, j * KEYS, r.limit, lane);
                if (st.due(j)) st.raise(st.highest(s), p.scale2, lane);
                const float ref = st.reference();
#pragma unroll
                for (int n = 0; n < 4; n++) pr[n] = st.exponentials(s, n, p.scale2, ref);
                stand(slot);
#pragma unroll
                for (int i = 0; i < AHEAD && i < VALUES; i++) read(i);
            }
            if (!late) copies.wait_for_next(j);
            phase_ends();
            if (DP > 96) __builtin_amdgcn_s_setprio(1);  // (16384 tokens, 8 heads of 128 930 -> 916 us; 8192 tokens, 16 heads of 96 379 -> 382)
            if (here) {
                multiply(FIRST, SCORES);
                if ((j + 1) * KEYS < wave_most) multiply(SCORES, END);
            }
            if (DP > 96) __builtin_amdgcn_s_setprio(0);
            if (late) {
                if (j + 1 == steps) break;
                copies.wait_for_next(j + 1);
            }
            phase_ends();
        }
        // Once more, and key by key where rows do not see all keys, if there turns out to be a NaN: rows that see none of its causes have none then
        int *flags = (int *)(lds + 2 * STAGES * H::TILE);
        const bool nan = st.doubtful(p.causal, p.D, lane);
        if (lane == 0) flags[wave] = nan;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int i = 0; i < WAVES; i++) any |= flags[i];
        careful = __builtin_amdgcn_readfirstlane(any) != 0;
        if (careful) {
            st.clear();
#pragma unroll 1
            for (int j = 0; j < steps; j++) {
                phase_ends();
                copies.ask_at(copies.first + j * copies.bytes, j, 0);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                phase_ends();
                if (j * KEYS >= wave_most) continue;
                score(0);
                const bool some = wave_least < (j + 1) * KEYS;
                if (some) hide(s, j * KEYS, r.limit, lane);
                st.attend_carefully(s, p.scale2, lds + STAGES * H::TILE, j * KEYS, r.limit, some, lane);
            }
        }
    }
    int row = wave0 + col;
    asm volatile("" : "+v"(row));  // (where the row goes is worked out anew: two registers through the loop are two too many)
    finish<BF16, H>(p, rows_of(p, it.r, hk, row), st, careful, lane);
}

// Adds the parts of every row (at most 64): four rows of a block per workgroup, a wave to a row, two columns per lane, 16 parts asked for at once; lane i holds part i's
// share of the row.
template <bool BF16, int BLOCK_ROWS, int SIZE>
__global__ void __launch_bounds__(256) self_attention_join_kernel(Params p) {
    constexpr int SUBS = BLOCK_ROWS / 4, MOST = 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, sub = rest % SUBS;
    Item it;
    if constexpr (BLOCK_ROWS > 32) {
        // one wave finds the block for all four: with many workgroups the search is most of their instructions (8192 tokens, one head of 64 30.4 -> 28.9 us, 304 workgroups in
        // parts 34.3 -> 33.5; a single token to 4096 keys, 32 heads over 8 of 128, 13.3 -> 13.5)
        __shared__ Item found;
        if (wave == 0) {
            const Item first = part_of<BLOCK_ROWS, SIZE, true>(p, rest / SUBS, lane);
            if (lane == 0) found = first;
        }
        __syncthreads();
        it.r = in_lane(found.r, 0);
        it.rb = __builtin_amdgcn_readfirstlane(found.rb);
        it.parts = __builtin_amdgcn_readfirstlane(found.parts);
        it.index = __builtin_amdgcn_readfirstlane(found.index);
        it.next = __builtin_amdgcn_readfirstlane(found.next);
        it.any = __builtin_amdgcn_readfirstlane((int)found.any) != 0;
    } else {
        it = part_of<BLOCK_ROWS, SIZE, true>(p, rest / SUBS, lane);
    }
    if (!it.any || it.parts == 1 || (long long)it.index + (long long)(it.parts - 1) * it.next >= p.items) return;
    const int at = sub * 4 + wave;
    const Rows r = rows_of(p, it.r, hk, it.rb * BLOCK_ROWS + at);
    if (!r.in) return;
    int least, most;
    limits_of(p, r, it.rb * BLOCK_ROWS, BLOCK_ROWS, least, most);
    it.parts = __popcll(__ballot(lane < it.parts && first_step<SIZE>(it, lane) * SIZE < most));  // (those that `share` has something for, but the first)
    if (it.parts < 2) return;
    const int c = lane * 2 < p.D ? lane * 2 : 0;
    typedef float float2_t __attribute__((ext_vector_type(2)));
    float top = -__builtin_huge_valf(), sum = 0.f;
    if (lane < it.parts) {
        const float2_t t = *(const float2_t *)stats_of<BLOCK_ROWS>(p, it.index + lane * it.next, hk, at);
        top = t[0];
        sum = t[1];
    }
    float x = 0.f, y = 0.f, f = 0.f;
    for (int first = 0; first < it.parts; first += MOST) {
        float2_t part[MOST];
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            part[i] = float2_t{0.f, 0.f};
            if (first + i < it.parts) part[i] = *(const float2_t *)(share_of<BLOCK_ROWS>(p, it.index + (first + i) * it.next, hk, at) + c);
        }
        if (first == 0) {
            float most = top;
#pragma unroll
            for (int d = 32; d; d >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, d));
            f = __builtin_amdgcn_exp2f(top - (most == -__builtin_huge_valf() ? 0.f : most));
            sum *= f;
#pragma unroll
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        }
#pragma unroll
        for (int i = 0; i < MOST; i++) {  // (zero times zero behind the last part)
            const float g = bits_f32(__builtin_amdgcn_readlane(f32_bits(f), first + i));
            x = __builtin_fmaf(part[i][0], g, x);
            y = __builtin_fmaf(part[i][1], g, y);
        }
    }
    const float inv = inverse(sum);
    if (lane * 2 < p.D) *(uint32_t *)(r.out + c * 2) = Elem<BF16>::pair(x * inv, y * inv);
}

enum Form { BY_KEYS, BY_ROWS, BY_TURNS };  // (keys in parts: the first two alone)

template <bool BF16, int DP, bool ONES>
int launch_kernels(const Params &p, Form form, hipStream_t st) {
    const int lds = form == BY_KEYS ? 8 * Head<DP, true>::TILE : form == BY_ROWS ? 4 * Head<DP>::TILE + 16 : 2 * STAGES * Head<DP>::TILE + 64;
    static bool reserved[3][64] = {{false}};
    const void *kernel = form == BY_KEYS ? (const void *)self_attention_keys_kernel<BF16, DP> : (const void *)self_attention_rows_kernel<BF16, DP, ONES>;
    if constexpr (DP > 64) {
        if (form == BY_TURNS) kernel = (const void *)self_attention_turns_kernel<BF16, DP, ONES>;
    }
    if (int rc = reserve_lds(kernel, lds, reserved[form], "self_attention")) return rc;
    const dim3 grid((unsigned)((long long)p.items * p.Hkv));
    if (form == BY_KEYS) SVDQ_LAUNCH((self_attention_keys_kernel<BF16, DP>), grid, dim3(256), lds, st, p);
    else if (form == BY_ROWS) SVDQ_LAUNCH((self_attention_rows_kernel<BF16, DP, ONES>), grid, dim3(256), lds, st, p);
    if constexpr (DP > 64) {
        if (form == BY_TURNS) SVDQ_LAUNCH((self_attention_turns_kernel<BF16, DP, ONES>), grid, dim3(64 * WAVES), lds, st, p);
    }
    int rc = check_launch("self_attention");
    if (rc || !p.target) return rc;
    if (form == BY_KEYS) SVDQ_LAUNCH((self_attention_join_kernel<BF16, 32, 32>), dim3((unsigned)(p.blocks * 8 * p.Hkv)), dim3(256), 0, st, p);
    else SVDQ_LAUNCH((self_attention_join_kernel<BF16, HALF, KEYS>), dim3((unsigned)(p.blocks * (HALF / 4) * p.Hkv)), dim3(256), 0, st, p);
    return check_launch("self_attention");
}

template <bool BF16, int DP>
int launch_head(const Params &p, Form form, hipStream_t st) {
    if (p.D < 32 * Head<DP>::DB) return launch_kernels<BF16, DP, true>(p, form, st);
    if constexpr (DP % 32 == 0) return launch_kernels<BF16, DP, false>(p, form, st);
    return SVDQ_EUNSUPPORTED;  // (not reached: the blocks of 80 end at 96)
}
template <bool BF16>
int launch_heads(const Params &p, Form form, hipStream_t st) {
    if (p.D <= 32) return launch_head<BF16, 32>(p, form, st);
    if (p.D <= 64) return launch_head<BF16, 64>(p, form, st);
    if (p.D <= 80) return launch_head<BF16, 80>(p, form, st);
    if (p.D <= 96) return launch_head<BF16, 96>(p, form, st);
    return launch_head<BF16, 128>(p, form, st);
}

struct Plan {
    Form form;
    long long blocks, items, target, least, mirror, workspace;
};

long long blocks_of(const svdq_self_attention_args *a, long long size) {
    const long long rows = a->q_len * (a->heads / a->kv_heads);
    // packed sequences: each, and the rows in front of them and behind, may end in the middle of a block
    return a->cu_seqlens_q ? rows / size + a->batch + 2 : (rows + size - 1) / size * a->batch;
}

// Which form a call takes and into how many parts it divides the keys of an average sequence: the least time by a model of the busiest compute unit, us.  Its constants are
// those of 252 shapes (heads of 32 to 128, 1 .. 8192 queries, causal or not), each in every form and 1 .. 32 parts; what it chooses is 1 to 2 % behind the fastest on average,
// 27 % at most (1024 tokens, 32 heads over 8 of 32, causal, 14.3 us against 11.3).  Chosen / others, us: 4 x 64 tokens, 8 heads of 128 rows 6.4 / keys 7.9, turns 7.3; 1024 tokens,
// 32 heads over 8 of 128, causal rows 24.6 / keys 54, turns 29; 16384 tokens, 8 heads of 128 turns 863 / rows 961; single tokens of 4 sequences of 8192 keys, 32 heads over 8 of 128
// 29.6 in eight parts / 115 whole; 64 tokens behind 8192, 32 over 8 heads of 128 rows in 16 parts 24.4 / keys in four 38.7; 4096 tokens, 8 heads of 128, causal rows in two parts
// 62.9 / whole 74, turns 82.
// Sequences of other lengths than the average have parts in proportion; of a cache the average is what it has room for.  One model for bf16 and fp16, whose steps take 3 to 6 %
// more, and without the memory's rate: 100 single tokens over 8192 keys of two heads of 128, 840 MB, are 112 us by it and take 160 (in parts 168 or more).
struct Cost {
    int head_dim;                   // up to
    float keys_base, round;         // keys form: first and last; a round of four waves' 32 keys
    float rows_base, rows_step;     // rows form: the same; a step of 64 keys
    float turns_base, turns_step;   // turns form, which heads up to 64 never take: 8192 tokens, 16 heads of 64 307 us by turns, 300 by rows, causal 632 and 573; of 32 255 and 212 (maxima at every step)
    float join, join_bytes;         // parts: the second launch; bytes a us of their way there and back
};
constexpr Cost costs[] = {{64, 4.2f, 0.72f, 4.3f, 0.69f, 0.f, 0.f, 5.4f, 3.5e6f}, {96, 5.7f, 1.45f, 4.8f, 0.95f, 5.5f, 1.10f, 5.6f, 5.2e6f}, {128, 6.1f, 1.65f, 5.6f, 1.06f, 7.0f, 1.30f, 5.5f, 6.2e6f}};

Plan plan_of(const svdq_self_attention_args *a, int cus) {
    const long long S = a->batch, q = a->cu_seqlens_q ? (a->q_len + S - 1) / S : a->q_len, k = a->cu_seqlens_k ? (a->k_len + S - 1) / S : a->k_len;
    const long long rows = q * (a->heads / a->kv_heads);
    const Cost &c = a->head_dim <= 64 ? costs[0] : a->head_dim <= 96 ? costs[1] : costs[2];
    // of the keys that a whole row of scores would have, how many are seen
    const float seen = !a->causal ? 1.f : q <= k ? 1.f - (float)(q - 1) / (2.f * (float)k) : (float)(k + 1) / (2.f * (float)q);
    const bool even = seen > 0.95f;
    static const int shares[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    Plan plan = {BY_TURNS, 0, 0, 0, 0, 0, 0};
    long long chosen = 1;
    float best = 0.f;
    for (int form = BY_KEYS; form <= (a->head_dim > 64 ? BY_TURNS : BY_ROWS); form++) {
        const int size = form == BY_KEYS ? 32 : form == BY_ROWS ? HALF : ROWS, step = form == BY_KEYS ? 32 : KEYS;
        const long long groups = (rows + size - 1) / size * S * a->kv_heads, steps = (k + step - 1) / step;
        for (int parts : shares) {
            if (parts > 1 && (form == BY_TURNS || S + 2 > MAX_REGIONS || groups * parts > 4 * cus || steps < (form == BY_KEYS ? 4 : 1) * parts)) break;
            const float w = (float)(groups * parts), each = (float)((steps + parts - 1) / parts), n = (float)cus;
            float t;
            if (form == BY_KEYS) {
                // two workgroups to a compute unit with heads up to 64, one with wider ones (LDS)
                const float slots = a->head_dim <= 64 ? 2.f * n : n, work = __builtin_ceilf(each / 4.f) * c.round * (w > n && a->head_dim <= 64 && even ? 1.3f : 1.f);
                t = c.keys_base + work;
                if (w > slots) {
                    const float more = (c.keys_base + work * seen) * (even ? __builtin_ceilf(w / slots) : w / slots + 0.3f);
                    t = more > t ? more : t;
                }
            } else {
                const float load = even ? __builtin_ceilf(w / n) : w * seen / n, turns = w / n < 1.f ? 1.f : w / n > 3.f ? 3.f : w / n;
                t = form == BY_ROWS ? c.rows_base + each * c.rows_step * (load > 1.f ? load : 1.f) : c.turns_base * turns + each * c.turns_step * (load > 1.f ? load : 1.f);
            }
            if (parts > 1) t += c.join + (float)(S * a->kv_heads * rows) * (float)(a->head_dim * 8) * (1.f + (float)(parts - 1) * seen) / c.join_bytes;
            if (best == 0.f || t < best) {
                best = t;
                chosen = parts;
                plan.form = (Form)form;
            }
        }
    }
    const int size = plan.form == BY_KEYS ? 32 : plan.form == BY_ROWS ? HALF : ROWS;
    // A compute unit gets its first workgroup and one of the second round at once.  With a causal mask the first have the most keys: those of the second round then come in the
    // opposite order, the longest with the shortest (4096 tokens, 8 heads of 128, causal, in two parts 75.6 -> 64.5 us; 16384, 2 heads of 64 155 -> 119).  Not where all have
    // about the same keys (chunks of new tokens behind long caches 34 -> 42), or where more rounds follow, which are given out as compute units come free (8 x 512 tokens, 32 heads over 8
    // of 128 35.1 -> 36.8).
    if (plan.form == BY_ROWS && !even && (rows + size - 1) / size * S * a->kv_heads * chosen <= 3 * cus) plan.mirror = cus / a->kv_heads;
    plan.blocks = plan.items = blocks_of(a, size);
    if (chosen > 1) {
        plan.least = plan.form == BY_KEYS ? 4 : 1;
        plan.target = (rows + size - 1) / size * S * chosen;
        plan.items = plan.blocks + plan.target + 1;
        plan.workspace = plan.items * a->kv_heads * size * (a->head_dim + 2) * 4;
    }
    return plan;
}

int check_args(const svdq_self_attention_args *a) {
    SVDQ_REQUIRE(a && a->q && a->k && a->v && a->out, "self_attention: q, k, v and out must not be null");
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "self_attention: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", (int)a->dtype);
    SVDQ_REQUIRE(a->batch > 0 && a->batch < 65536 && a->heads > 0 && a->heads < 65536 && a->kv_heads > 0 && a->heads % a->kv_heads == 0,
                 "self_attention: batch (%lld) and heads (%lld) must be in 1..65535, kv_heads (%lld) must divide heads", (long long)a->batch, (long long)a->heads, (long long)a->kv_heads);
    SVDQ_REQUIRE(a->head_dim > 0 && a->head_dim <= 128 && a->head_dim % 8 == 0, "self_attention: head_dim (%lld) must be a multiple of 8 up to 128", (long long)a->head_dim);
    SVDQ_REQUIRE(a->q_len > 0 && a->k_len > 0 && a->k_len < (1ll << 31) - 512, "self_attention: q_len (%lld) and k_len (%lld) must be positive, k_len below 2^31 - 512", (long long)a->q_len,
                 (long long)a->k_len);
    SVDQ_REQUIRE(a->q_len < (1ll << 31) && a->q_len * (a->heads / a->kv_heads) < (1ll << 31) - 512,
                 "self_attention: q_len (%lld) times the heads that share keys must be below 2^31 - 512", (long long)a->q_len);
    // (a launch takes fewer than 2^32 threads, 256 for 32 rows at most)
    SVDQ_REQUIRE(blocks_of(a, 32) < (1ll << 24) && blocks_of(a, 32) * a->kv_heads < (1ll << 24), "self_attention: %lld queries of %lld heads are too many for one launch", (long long)a->q_len,
                 (long long)a->heads);
    SVDQ_REQUIRE(!a->key_lengths || !a->cu_seqlens_k, "self_attention: at most one of key_lengths and cu_seqlens_k can be given");
    SVDQ_REQUIRE(a->scale > 0.f && a->scale < __builtin_huge_valf(), "self_attention: scale must be a positive number");
    for (int i = 0; i < 3; i++)
        SVDQ_REQUIRE(a->q_stride[i] >= 0 && a->k_stride[i] >= 0 && a->v_stride[i] >= 0 && a->out_stride[i] >= 0 &&
                         (a->q_stride[i] | a->k_stride[i] | a->v_stride[i] | a->out_stride[i]) % 8 == 0,
                     "self_attention: strides must be multiples of 8 elements (16 bytes)");
    SVDQ_REQUIRE(a->k_stride[1] < (1ll << 24) && a->v_stride[1] < (1ll << 24), "self_attention: the tokens of k and v must be less than 2^24 elements apart");
    SVDQ_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)a->workspace) % 16 == 0, "self_attention: pointers must be 16-byte aligned");
    SVDQ_REQUIRE(((uintptr_t)a->key_lengths | (uintptr_t)a->cu_seqlens_q | (uintptr_t)a->cu_seqlens_k) % 4 == 0,
                 "self_attention: key_lengths, cu_seqlens_q and cu_seqlens_k must be 4-byte aligned");
    return SVDQ_OK;
}

int current_compute_units(int &cus) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || (cus = compute_units(dev)) == 0) {
        (void)hipGetLastError();
        return fail(SVDQ_ELAUNCH, "self_attention: no current device");
    }
    return SVDQ_OK;
}

}  // namespace

extern "C" int svdq_self_attention_workspace(const svdq_self_attention_args *a, int64_t *bytes) {
    if (int rc = check_args(a)) return rc;
    SVDQ_REQUIRE(bytes, "self_attention: bytes must not be null");
    int cus;
    if (int rc = current_compute_units(cus)) return rc;
    *bytes = plan_of(a, cus).workspace;
    return SVDQ_OK;
}

extern "C" int svdq_self_attention(const svdq_self_attention_args *a, void *stream) {
    if (int rc = check_args(a)) return rc;
    int cus;
    if (int rc = current_compute_units(cus)) return rc;
    const Plan plan = plan_of(a, cus);
    SVDQ_REQUIRE(plan.workspace == 0 || (a->workspace && a->workspace_bytes >= plan.workspace), "self_attention: needs a workspace of %lld bytes, got %lld", plan.workspace,
                 (long long)(a->workspace ? a->workspace_bytes : 0));
    Params p;
    p.q = (const char *)a->q;
    p.k = (const char *)a->k;
    p.v = (const char *)a->v;
    p.out = (char *)a->out;
    p.cu_q = a->cu_seqlens_q;
    p.cu_k = a->cu_seqlens_k;
    p.lengths = a->key_lengths;
    p.partial = (float *)a->workspace;
    for (int i = 0; i < 3; i++) {
        p.qs[i] = a->q_stride[i] * 2;
        p.ks[i] = a->k_stride[i] * 2;
        p.vs[i] = a->v_stride[i] * 2;
        p.os[i] = a->out_stride[i] * 2;
    }
    p.S = (int)a->batch;
    p.Hkv = (int)a->kv_heads;
    p.G = (int)(a->heads / a->kv_heads);
    p.D = (int)a->head_dim;
    p.Tq = (int)a->q_len;
    p.Tk = (int)a->k_len;
    p.items = (int)plan.items;
    p.blocks = (int)plan.blocks;
    p.target = (int)plan.target;
    p.least = (int)plan.least;
    p.mirror = (int)plan.mirror;
    p.causal = a->causal != 0;
    p.zero_rest = a->zero_rest != 0;
    p.scale2 = a->scale * 1.44269504088896340736f;
    return a->dtype == SVDQ_BF16 ? launch_heads<true>(p, plan.form, (hipStream_t)stream) : launch_heads<false>(p, plan.form, (hipStream_t)stream);
}
