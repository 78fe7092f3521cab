// out[m][n] = T(float(sum_k act[m][k] * wgt[n][k]) * (ascales[m] * wscales[n]) + bias[n]) on v_mfma_i32_32x32x32_i8 /
// v_mfma_i32_16x16x64_i8.  The integer sums are exact, whatever their order; each factor, the product with it, the bias and the
// result are rounded once.
#include "svdq_common.h"

using namespace svdq;

namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int int16_t_ __attribute__((ext_vector_type(16)));

struct W8A8Params {
    const char *act, *wgt;
    const float *ascales, *wscales;
    const uint16_t *bias;
    uint16_t *out;
    long long ld_act, ld_wgt, ld_out;  // bytes, bytes, elements
    int M, N, K, bf16;
    int tiles_m, tiles_n;
    int parts;          // along K; with more than one, a workgroup leaves its sums in `partial` and a small kernel finishes
    int *partial;       // [part][M][ld_partial]
    long long ld_partial;
    int wide;  // rows of `out` and its first column are 16 bytes apart and aligned
};

// What copies of a piece behind a row's end read.
__device__ const u32x4_t zeros16 = {0, 0, 0, 0};

__device__ inline float value16(uint16_t b, int bf16) { return bf16 ? bf16_bits_to_f32(b) : (float)__builtin_bit_cast(_Float16, b); }
__device__ inline uint32_t pair16(float lo, float hi, int bf16) {
    if (bf16) return pack_bf16x2(lo, hi);
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}

// Workgroup -> tile.  Workgroups go round robin over the 8 XCDs, each with an L2 of its own: an XCD gets one contiguous run of the
// tiles, which are numbered down the rows inside bands of up to BAND row blocks, so that the tiles at work on an XCD share operands.
constexpr int BAND = 8;
__device__ inline void tile_of(const W8A8Params &p, int &tm, int &tn) {
    const int total = p.tiles_m * p.tiles_n, id = blockIdx.x;  // (of the part blockIdx.y)
    const int xcd = id & 7, per = total >> 3, more = total & 7;
    const int tile = xcd * per + (xcd < more ? xcd : more) + (id >> 3);
    const int band_tiles = BAND * p.tiles_n, band = tile / band_tiles, in = tile - band * band_tiles;
    const int height = p.tiles_m - band * BAND < BAND ? p.tiles_m - band * BAND : BAND;
    tm = band * BAND + in % height;
    tn = in / height;
}

// ---- tiles through LDS --------------------------------------------------------------------------------------------------
// BM x BN outputs by WM x WN waves.  128 bytes of K of every row make a stage of the ring; they come by asynchronous copies of
// 16 bytes a lane, a KB (8 rows) a request.  Piece p of row r stands at place p ^ ((r / 2) % 8) of its row: 16 lanes that read the
// same piece of 16 rows then touch every bank once.  The weights are the left operand, so that a lane holds four consecutive
// columns of one row.  Bound, for the large ones, by the power limit: 8192 x 8192 x 8192 471 us, 2335 TOP/s (353 us on zeros); the 256 x 256 tile's step of 128 of K
// is 2048 cycles of a SIMD's matrix instructions next to 1024 of copies and 840 of reads from LDS.  By four waves of 128 x 128, which read a third less,
// but are alone on their SIMDs, it takes 698.
constexpr int BK = 128;
__device__ inline int swizzle(int row) { return (row >> 1) & 7; }

template <int BM, int BN, int WM, int WN, int STAGES>
struct Tiles {
    static constexpr int THREADS = WM * WN * 64, WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    static constexpr int A_REQ = BM / 8 / WAVES, B_REQ = BN / 8 / WAVES, REQ = A_REQ + B_REQ;
    static constexpr int STAGE = (BM + BN) * BK, LDS = STAGE * STAGES;
    static constexpr int SLAB_LD = TN * 32 + 8;  // elements
    static_assert(WAVES * 32 * SLAB_LD * 2 <= LDS, "the epilogue's slabs reuse the ring");
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "");
};

template <int BM, int BN, int WM, int WN, int STAGES, int OCC>
__global__ void __launch_bounds__(WM *WN * 64, OCC) w8a8_tiles_kernel(W8A8Params p) {
    using T = Tiles<BM, BN, WM, WN, STAGES>;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int tm, tn;
    tile_of(p, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    // copies: request i of this wave brings rows (wave * REQ + i) * 8 + lane / 8; rows behind the last are the last again
    const int sub = lane >> 3;
    const char *src_a = p.act + (long long)m0 * p.ld_act, *src_b = p.wgt + (long long)n0 * p.ld_wgt;
    uint32_t off_a[T::A_REQ], off_b[T::B_REQ];
    auto piece = [&](int row) __attribute__((always_inline)) { return ((lane & 7) ^ swizzle(row)) * 16; };
#pragma unroll
    for (int i = 0; i < T::A_REQ; i++) {
        const int r = (wave * T::A_REQ + i) * 8 + sub, last = p.M - 1 - m0;
        off_a[i] = (uint32_t)((r < last ? r : last) * p.ld_act) + piece(r);
    }
#pragma unroll
    for (int i = 0; i < T::B_REQ; i++) {
        const int r = (wave * T::B_REQ + i) * 8 + sub, last = p.N - 1 - n0;
        off_b[i] = (uint32_t)((r < last ? r : last) * p.ld_wgt) + piece(r);
    }
    // this part's steps along K
    const int whole = p.K / BK, all = (p.K + BK - 1) / BK;
    const int begin = (int)((long long)all * blockIdx.y / p.parts), steps = (int)((long long)all * (blockIdx.y + 1) / p.parts) - begin;
    const uint32_t dst_a = base + wave * T::A_REQ * 1024, dst_b = base + BM * BK + wave * T::B_REQ * 1024;
    auto request = [&](int n) __attribute__((always_inline)) {
        const uint32_t stage = (uint32_t)(n % STAGES) * T::STAGE;
        const int step = begin + n;
        const char *a = src_a + (long long)step * BK, *b = src_b + (long long)step * BK;
        if (step < whole) {
#pragma unroll
            for (int i = 0; i < T::A_REQ; i++)
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst_a + stage + i * 1024), "v"(off_a[i]), "s"(a) : "memory", "m0");
#pragma unroll
            for (int i = 0; i < T::B_REQ; i++)
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst_b + stage + i * 1024), "v"(off_b[i]), "s"(b) : "memory", "m0");
        } else {  // the last, partly filled step: zeros behind the row's end
            const int left = p.K - step * BK;
#pragma unroll
            for (int i = 0; i < T::A_REQ; i++) {
                const char *s = piece((wave * T::A_REQ + i) * 8 + sub) < left ? a + off_a[i] : (const char *)&zeros16;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst_a + stage + i * 1024), "v"(s) : "memory", "m0");
            }
#pragma unroll
            for (int i = 0; i < T::B_REQ; i++) {
                const char *s = piece((wave * T::B_REQ + i) * 8 + sub) < left ? b + off_b[i] : (const char *)&zeros16;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst_b + stage + i * 1024), "v"(s) : "memory", "m0");
            }
        }
    };
    // Eight waves are two on every SIMD: the second four ask for their copies behind their first matrix instructions, while the first four,
    // which do it in front, are still at it (8192 x 8192 x 8192: 481 -> 475 us; with one wave each it costs up to 10 %)
    const bool late = BM == 256 && BN == 256 && wave >= T::WAVES / 2;
    int16_t_ acc[T::TM][T::TN];
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
        for (int j = 0; j < T::TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
        if (s < steps) request(s);
    const int col = lane & 31, h = lane >> 5;
    const char *row_a = lds + (wm * T::TM * 32 + col) * BK, *row_b = lds + BM * BK + (wn * T::TN * 32 + col) * BK;
    for (int step = 0; step < steps; step++) {
        // this step's copies have landed (of all waves), and nobody reads the stage that the next request overwrites
        if (step + STAGES - 1 <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * T::REQ) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int stage = (step % STAGES) * T::STAGE;
        // operands of one 32 of K ahead of the matrix instructions; the copies are asked for behind the first ones
        int4_t a[2][T::TM], b[2][T::TN];
        auto read = [&](int ks) __attribute__((always_inline)) {
            const int at = ((2 * ks + h) ^ swizzle(col)) * 16;
#pragma unroll
            for (int i = 0; i < T::TM; i++) a[ks & 1][i] = *(const int4_t *)(row_a + stage + i * 32 * BK + at);
#pragma unroll
            for (int j = 0; j < T::TN; j++) b[ks & 1][j] = *(const int4_t *)(row_b + stage + j * 32 * BK + at);
        };
        read(0);
        __builtin_amdgcn_sched_barrier(0);
        const bool more = step + STAGES - 1 < steps;
        if (more && !late) request(step + STAGES - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < BK / 32; ks++) {
            if (ks + 1 < BK / 32) read(ks + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < T::TM; i++)
#pragma unroll
                for (int j = 0; j < T::TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[ks & 1][j], a[ks & 1][i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (BM == 256 && BN == 256 && ks == 0 && more && late) request(step + STAGES - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (p.parts > 1) {
        int *part = p.partial + (long long)blockIdx.y * p.M * p.ld_partial;
#pragma unroll
        for (int i = 0; i < T::TM; i++) {
            const int row = m0 + (wm * T::TM + i) * 32 + col;
#pragma unroll
            for (int j = 0; j < T::TN; j++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int n = n0 + (wn * T::TN + j) * 32 + 8 * g + 4 * h;
                    if (row < p.M && n < p.ld_partial)
                        *(int4_t *)(part + row * p.ld_partial + n) = int4_t{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                }
        }
        return;
    }
    // epilogue: 32 rows at a time through the wave's slab in LDS, in the place of the ring
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    uint16_t *slab = (uint16_t *)lds + wave * 32 * T::SLAB_LD;
    const int wave_n = n0 + wn * T::TN * 32;
#pragma unroll
    for (int i = 0; i < T::TM; i++) {
        const int row0 = m0 + (wm * T::TM + i) * 32, row = row0 + col;
        const float sa = row < p.M ? p.ascales[row] : 0.f;
#pragma unroll
        for (int j = 0; j < T::TN; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int c = j * 32 + 8 * g + 4 * h, n = wave_n + c;
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int ne = n + e < p.N ? n + e : p.N - 1;
                    y[e] = (float)acc[i][j][4 * g + e] * (sa * p.wscales[ne]);
                    if (p.bias) y[e] += value16(p.bias[ne], p.bf16);
                }
                *(u32x2_t *)(slab + col * T::SLAB_LD + c) = u32x2_t{pair16(y[0], y[1], p.bf16), pair16(y[2], y[3], p.bf16)};
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (p.wide) {
            constexpr int LANES = T::TN * 4, PER = 64 / LANES;  // lanes per row, rows per pass
#pragma unroll
            for (int r = 0; r < 32; r += PER) {
                const int rr = r + lane / LANES, cc = (lane % LANES) * 8;
                const u32x4_t v = *(const u32x4_t *)(slab + rr * T::SLAB_LD + cc);
                if (row0 + rr < p.M && wave_n + cc < p.N) __builtin_nontemporal_store(v, (u32x4_t *)(p.out + (row0 + rr) * p.ld_out + wave_n + cc));
            }
        } else {
            for (int e = lane; e < 32 * T::TN * 32; e += 64) {
                const int rr = e / (T::TN * 32), cc = e % (T::TN * 32);
                if (row0 + rr < p.M && wave_n + cc < p.N) p.out[(row0 + rr) * p.ld_out + wave_n + cc] = slab[rr * T::SLAB_LD + cc];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// 16 columns x 16 rows per workgroup, whose WAVES waves split K in steps of 64 bytes and meet in LDS.  Operands go from memory to the
// registers of the wave that multiplies them.  Bound by the weights' way from memory: 1 x 4096 x 12288 12 us, 4.1 TB/s with the launch.
template <int WAVES>
__global__ void __launch_bounds__(WAVES * 64) w8a8_few_rows_kernel(W8A8Params p) {
    __shared__ int4_t sums[WAVES - 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16;
    const char *w = p.wgt + (long long)(n0 + r < p.N ? n0 + r : p.N - 1) * p.ld_wgt + q * 16;
    const char *a = p.act + (long long)(r < p.M ? r : p.M - 1) * p.ld_act + q * 16;
    int4_t acc = int4_t{0, 0, 0, 0};
    // this part's steps of 64 bytes, in turns of UN: the waves take them one after the other (UN = 4: 1 x 4096 x 12288 13.3 us against 12.2,
    // 1 x 4096 x 4096 7.9 against 7.3; 8: 12.4 and 7.5 with eight waves)
    constexpr int UN = 2;
    const int whole = p.K / 64, turns = ((p.K + 63) / 64 + UN - 1) / UN;
    const int first = (int)((long long)turns * blockIdx.y / p.parts), last = (int)((long long)turns * (blockIdx.y + 1) / p.parts);
    int s = (first + wave) * UN;
    for (; s + UN <= whole && s < last * UN; s += WAVES * UN) {
        int4_t wv[UN], av[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            wv[u] = *(const int4_t *)(w + (s + u) * 64);
            av[u] = *(const int4_t *)(a + (s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < UN; u++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u], av[u], acc, 0, 0, 0);
    }
    // (the wave whose turn holds the last whole steps and the partly filled one)
    for (; s * 64 < p.K && s < last * UN; s++) {
        const bool in = s * 64 + q * 16 < p.K;
        int4_t wv = int4_t{0, 0, 0, 0}, av = int4_t{0, 0, 0, 0};
        if (in) {
            wv = *(const int4_t *)(w + s * 64);
            av = *(const int4_t *)(a + s * 64);
        }
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, av, acc, 0, 0, 0);
        if ((s + 1) % UN == 0) break;
    }
    if (wave > 0) sums[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0 || r >= p.M) return;
#pragma unroll
    for (int v = 0; v < WAVES - 1; v++) acc += sums[v][lane];
    // four consecutive columns of row r
    const int n = n0 + 4 * q;
    if (p.parts > 1) {
        if (n < p.ld_partial) *(int4_t *)(p.partial + ((long long)blockIdx.y * p.M + r) * p.ld_partial + n) = acc;
        return;
    }
    const float sa = p.ascales[r];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= p.N) break;
        float y = (float)acc[e] * (sa * p.wscales[n + e]);
        if (p.bias) y += value16(p.bias[n + e], p.bf16);
        p.out[r * p.ld_out + n + e] = (uint16_t)pair16(y, 0.f, p.bf16);
    }
}

// ---- the parts' sums, scales and bias: four columns per thread -----------------------------------------------------------------
__global__ void __launch_bounds__(256) w8a8_join_kernel(W8A8Params p) {
    const int n = (blockIdx.x * 64 + (threadIdx.x & 63)) * 4, m = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (n >= p.N || m >= p.M) return;
    const int *src = p.partial + m * p.ld_partial + n;
    int4_t acc = *(const int4_t *)src;
    for (int i = 1; i < p.parts; i++) acc += *(const int4_t *)(src + (long long)i * p.M * p.ld_partial);
    const float sa = p.ascales[m];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int ne = n + e < p.N ? n + e : p.N - 1;
        y[e] = (float)acc[e] * (sa * p.wscales[ne]);
        if (p.bias) y[e] += value16(p.bias[ne], p.bf16);
    }
    uint16_t *out = p.out + m * p.ld_out + n;
    const u32x2_t w = {pair16(y[0], y[1], p.bf16), pair16(y[2], y[3], p.bf16)};
    if (p.wide) {
        *(u32x2_t *)out = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < p.N) out[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
}

int join(const W8A8Params &p, hipStream_t st) {
    int rc = check_launch("gemm_w8a8");
    if (rc || p.parts == 1) return rc;
    SVDQ_LAUNCH(w8a8_join_kernel, dim3((unsigned)((p.N + 255) / 256), (unsigned)((p.M + 3) / 4)), dim3(256), 0, st, p);
    return check_launch("gemm_w8a8");
}

template <int BM, int BN, int WM, int WN, int STAGES, int OCC>
int launch_tiles(W8A8Params &p, hipStream_t st) {
    using T = Tiles<BM, BN, WM, WN, STAGES>;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    if ((long long)p.tiles_m * p.tiles_n * T::THREADS >= (1ll << 32)) return fail(SVDQ_EUNSUPPORTED, "gemm_w8a8: %d x %d tiles are too many for one launch", p.tiles_m, p.tiles_n);
    auto *kernel = w8a8_tiles_kernel<BM, BN, WM, WN, STAGES, OCC>;
    static bool reserved[64] = {false};
    if (int rc = reserve_lds((const void *)kernel, T::LDS, reserved, "gemm_w8a8")) return rc;
    SVDQ_LAUNCH(kernel, dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.parts), dim3(T::THREADS), T::LDS, st, p);
    return join(p, st);
}

template <int WAVES>
int launch_few(W8A8Params &p, hipStream_t st) {
    SVDQ_LAUNCH((w8a8_few_rows_kernel<WAVES>), dim3((unsigned)((p.N + 15) / 16), (unsigned)p.parts), dim3(WAVES * 64), 0, st, p);
    return join(p, st);
}

// ---- which kernel ----------------------------------------------------------------------------------------------------------------
enum Form { FEW_4, FEW_8, T32x64, T64x64_DEEP, T64x64, T64x128, T128x128, T256x256 };
struct Plan {
    Form form;
    int parts;
    long long workspace;
};

// A model of the busiest compute unit's time, in us, fitted to 32 shapes of 17 .. 16384 rows (each form and number of parts timed; what it
// chooses is 0.8 % behind the fastest on average, 13 % at most): a step of 128 bytes of K takes a workgroup `alone` while it has its compute
// unit to itself and every one of several `share`; `slots` fit a compute unit.  A tile ends with its output's way to memory (20 bytes a ns for a
// compute unit when all write) and 0.4 us of latencies; the kernel that joins parts takes 1.4 us and its traffic.  Few rows are the weights'
// way from memory.
// Chosen / next best form, us: 505 x 2304 x 4608 14.3 (64 x 64) / 15.9, 256 x 4096 x 4096 14.7 (64 x 64, four stages) / 16.1, 1024 x 4096 x 4096 28.1
// (64 x 128) / 29.2, 2048 x 4096 x 4096 38.1 (128 x 128) / 51.1, 7747 x 13984 x 156 46.6 (128 x 128 in four parts; whole 89.8), 17 x 13728 x 3213 14.3
// (32 x 64 in five parts; whole 33.1), 4608 x 4096 x 16384 306 (256 x 256) / 335.  Tiles of 128 x 256 in three stages were ahead at 3 of the shapes
// only, those with the most operand bytes for a round of tiles (1024 x 8192 x 8192 72.3 / 79.1), behind at the others (2048 x 4096 x 4096 41.5).  64 x 128
// by eight waves instead of four: 512 x 4096 x 4096 18.3 / 20.2, 1300 x 2304 x 1152 12.1 / 13.8, 1157 x 2304 x 4608 26.8 / 28.7; 128 x 128 by four instead of
// eight 26.9 / 25.3 (3000 x 640 x 5120); 64 x 64 in three stages 15.5 / 15.0 (505 x 2304 x 4608).
struct Cost {
    Form form;
    int bm, bn, slots;
    float alone, share;
};
constexpr Cost costs[] = {
    {T32x64, 32, 64, 3, 0.235f, 0.205f},   {T64x64_DEEP, 64, 64, 2, 0.265f, 0.19f}, {T64x64, 64, 64, 5, 0.475f, 0.195f},
    {T64x128, 64, 128, 2, 0.36f, 0.325f}, {T128x128, 128, 128, 2, 0.65f, 0.455f},  {T256x256, 256, 256, 1, 1.48f, 1.48f},
};
constexpr int MAX_PARTS = 16;

Plan plan_of(long long M, long long N, long long K, int cus) {
    const long long steps = (K + BK - 1) / BK;
    Plan plan = {T256x256, 1, 0};
    const long long few = (N + 15) / 16;
    if (M <= 8 || (M <= 16 && few < 2 * cus)) {
        // 16 columns a workgroup: with few of them eight waves instead of four, and parts of at least two turns for each wave
        // (1 x 4096 x 4096 7.5 -> 7.3 us with eight waves, 8 x 16384 x 512 14.2 -> 9.2 in parts; 1 x 4096 x 12288 12.2 with four, 13.1 with
        // eight).  More than eight rows on many columns go to tiles, whose activations come once per 64 columns (16 x 4096 x 12288 15.1 -> 13.9;
        // eight rows 13.3 here, 13.1 there)
        const long long tiles = few, most = K / 2048, want = cus / tiles;
        plan.form = tiles >= 2 * cus ? FEW_4 : FEW_8;
        if (want > 1 && most > 1) plan.parts = (int)(want < most ? want : most);
        if (plan.parts > MAX_PARTS) plan.parts = MAX_PARTS;
    } else {
        float best = 0.f;
        for (const Cost &c : costs) {
            const long long tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
            const float last = c.bm * c.bn * 2 / 20000.f;  // a tile's output
            for (int parts = 1; parts <= MAX_PARTS && (parts == 1 || (steps >= 4 * parts && tiles * (parts - 1) < c.slots * cus)); parts++) {
                const long long most = (tiles * parts + cus - 1) / cus, rounds = most / c.slots, rest = most % c.slots;
                const float n = (float)((steps + parts - 1) / parts);
                auto round = [&](long long w) { return n * (c.alone > w * c.share ? c.alone : w * c.share) + 0.4f + w * last * (parts > 1 ? 2.f : 1.f); };
                float t = rounds * round(c.slots) + (rest ? round(rest) : 0.f);
                if (parts > 1) t += 1.4f + M * N * 4.f * parts / 4.0e6f;
                if (best == 0.f || t < best) {
                    best = t;
                    plan.form = c.form;
                    plan.parts = parts;
                }
            }
        }
    }
    plan.workspace = plan.parts > 1 ? plan.parts * M * ((N + 3) / 4 * 4) * 4 : 0;
    return plan;
}

int plan_call(const svdq_gemm_w8a8_args *a, Plan &plan) {
    SVDQ_REQUIRE(a && a->act && a->wgt && a->ascales && a->wscales && a->out, "gemm_w8a8: act, wgt, ascales, wscales and out must not be null");
    SVDQ_REQUIRE(a->dtype == SVDQ_BF16 || a->dtype == SVDQ_FP16, "gemm_w8a8: dtype must be SVDQ_BF16 or SVDQ_FP16, got %d", (int)a->dtype);
    SVDQ_REQUIRE(a->M > 0 && a->N > 0 && a->M < (1ll << 31) - 256 && a->N < (1ll << 28) - 256, "gemm_w8a8: M (%lld) must be positive and below 2^31 - 256, N (%lld) below 2^28 - 256",
                 (long long)a->M, (long long)a->N);
    // (a launch takes fewer than 2^32 threads: 128 to 512 a tile, 32 x 64 the smallest of them; 512 for 16 columns of few rows)
    SVDQ_REQUIRE(((a->M + 31) / 32) * ((a->N + 63) / 64) < (1ll << 24), "gemm_w8a8: %lld x %lld outputs are too many for one launch (2^24 tiles of 32 x 64)", (long long)a->M,
                 (long long)a->N);
    // 127 * 127 * 131072 and 128 * 128 * 131056 stay below 2^31
    SVDQ_REQUIRE(a->K > 0 && a->K % 16 == 0 && a->K < 131072, "gemm_w8a8: K (%lld) must be a multiple of 16 below 131072, so that the integer sums cannot overflow", (long long)a->K);
    SVDQ_REQUIRE(a->ld_act >= a->K && a->ld_act % 16 == 0 && a->ld_act < (1ll << 23), "gemm_w8a8: rows of act must be at least K bytes, a multiple of 16 and less than 2^23 apart, got %lld",
                 (long long)a->ld_act);
    SVDQ_REQUIRE(a->ld_wgt >= a->K && a->ld_wgt % 16 == 0 && a->ld_wgt < (1ll << 23), "gemm_w8a8: rows of wgt must be at least K bytes, a multiple of 16 and less than 2^23 apart, got %lld",
                 (long long)a->ld_wgt);
    SVDQ_REQUIRE(a->ld_out >= a->N, "gemm_w8a8: rows of out must be at least N (%lld) elements apart, got %lld", (long long)a->N, (long long)a->ld_out);
    SVDQ_REQUIRE(((uintptr_t)a->act | (uintptr_t)a->wgt | (uintptr_t)a->workspace) % 16 == 0, "gemm_w8a8: act, wgt and workspace must be 16-byte aligned");
    SVDQ_REQUIRE(((uintptr_t)a->ascales | (uintptr_t)a->wscales) % 4 == 0 && ((uintptr_t)a->bias | (uintptr_t)a->out) % 2 == 0, "gemm_w8a8: scales, bias and out must be aligned to their elements");
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || (cus = compute_units(dev)) == 0) {
        (void)hipGetLastError();
        return fail(SVDQ_ELAUNCH, "gemm_w8a8: no current device");
    }
    plan = plan_of(a->M, a->N, a->K, cus);
    return SVDQ_OK;
}

}  // namespace

extern "C" int svdq_gemm_w8a8_workspace(const svdq_gemm_w8a8_args *a, int64_t *bytes) {
    Plan plan;
    if (int rc = plan_call(a, plan)) return rc;
    SVDQ_REQUIRE(bytes, "gemm_w8a8: bytes must not be null");
    *bytes = plan.workspace;
    return SVDQ_OK;
}

extern "C" int svdq_gemm_w8a8(const svdq_gemm_w8a8_args *a, void *stream) {
    Plan plan;
    if (int rc = plan_call(a, plan)) return rc;
    SVDQ_REQUIRE(plan.workspace == 0 || (a->workspace && a->workspace_bytes >= plan.workspace), "gemm_w8a8: needs a workspace of %lld bytes, got %lld", plan.workspace,
                 (long long)(a->workspace ? a->workspace_bytes : 0));
    W8A8Params p;
    p.act = (const char *)a->act;
    p.wgt = (const char *)a->wgt;
    p.ascales = a->ascales;
    p.wscales = a->wscales;
    p.bias = (const uint16_t *)a->bias;
    p.out = (uint16_t *)a->out;
    p.ld_act = a->ld_act;
    p.ld_wgt = a->ld_wgt;
    p.ld_out = a->ld_out;
    p.M = (int)a->M;
    p.N = (int)a->N;
    p.K = (int)a->K;
    p.bf16 = a->dtype == SVDQ_BF16;
    p.wide = a->N % 8 == 0 && a->ld_out % 8 == 0 && (uintptr_t)a->out % 16 == 0;
    p.parts = plan.parts;
    p.ld_partial = (a->N + 3) / 4 * 4;
    p.partial = (int *)a->workspace;
    hipStream_t st = (hipStream_t)stream;
    switch (plan.form) {
    case FEW_4: return launch_few<4>(p, st);
    case FEW_8: return launch_few<8>(p, st);
    case T32x64: return launch_tiles<32, 64, 1, 2, 4, 2>(p, st);
    case T64x64_DEEP: return launch_tiles<64, 64, 2, 2, 4, 2>(p, st);
    case T64x64: return launch_tiles<64, 64, 2, 2, 2, 2>(p, st);
    case T64x128: return launch_tiles<64, 128, 2, 4, 3, 2>(p, st);
    case T128x128: return launch_tiles<128, 128, 4, 2, 2, 2>(p, st);
    default: return launch_tiles<256, 256, 2, 4, 2, 2>(p, st);
    }
}
