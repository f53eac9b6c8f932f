// Matrix products grouped by expert, 16-bit weights in their checkpoint layout.
//
//   y[r, n] = sum_k x[row(r), k] * W[e(r), n, k]          grouped_linear
//   h[r, i] = silu(sum x Wg) * (sum x Wu)                 grouped_gate_up
//
// Rows r come grouped by expert (offsets as moe_dispatch writes them); sums in
// fp32, one rounding when a value is stored. What the reference runs per token
// with fp32 experts (cuda/moe_expert.cu:32-130).
#include "grouped.hpp"

#include "num16.hpp"

namespace glmmoe {

// Row tiles (2^lg rows at most) of the groups off[0 .. E], and of group E, the shared expert's
// rows, where there is one: large tiles (more than 2^lg / 2 rows) in expert order, then small ones. Every
// wave calls it and gets the same answer. Offsets are clamped to [0, rows], so that no tile
// leaves the rows whatever they hold. Lane i looks after `per` consecutive experts.
struct TileScan {
    const GroupedArgs& a;
    int lg, per;
    int o[10];                                      // per <= 9: the lane's offsets
    int nbig, nsmall, ibig, ismall;                 // the lane's tiles, and up to and with its

    __device__ __forceinline__ int at(int i) const { return min(max(a.off[min(i, a.E)], 0), a.rows); }
    // f(expert, first row, rows) for the lane's experts.
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        const int e0 = (threadIdx.x & 63) * per;
        auto one = [&](int e, int lo, int hi) {
            if (e == a.E) lo = a.sh_row, hi = a.sh_row + a.sh_rows;
            f(e, lo, max(hi - lo, 0));
        };
        if (per <= 9) {
#pragma unroll
            for (int j = 0; j < 9; ++j)
                if (j < per) one(e0 + j, o[j], o[j + 1]);
        } else {
            for (int j = 0; j < per; ++j) one(e0 + j, at(e0 + j), at(e0 + j + 1));
        }
    }
    __device__ __forceinline__ int big(int n) const {
        return (n >> lg) + ((n & ((1 << lg) - 1)) > 1 << (lg - 1));
    }
    __device__ __forceinline__ int small(int n) const {
        const int rest = n & ((1 << lg) - 1);
        return rest > 0 && rest <= 1 << (lg - 1);
    }
    __device__ __forceinline__ TileScan(const GroupedArgs& a_, int lg_)
        : a(a_), lg(lg_), per((a_.E + 64) / 64), nbig(0), nsmall(0) {
        const int lane = threadIdx.x & 63;
        if (per <= 9) {
#pragma unroll
            for (int j = 0; j < 10; ++j)
                if (j <= per) o[j] = at(lane * per + j);
        }
        each([&](int, int, int n) { nbig += big(n), nsmall += small(n); });
        ibig = nbig, ismall = nsmall;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(ibig, d), v = __shfl_up(ismall, d);
            if (lane >= d) ibig += u, ismall += v;
        }
    }
    // Tile t of a class, found by the lane that has it.
    __device__ __forceinline__ bool find(bool large, int t, int& e, int& r0, int& nr) const {
        const int mine = large ? nbig : nsmall, incl = large ? ibig : ismall;
        const uint64_t past = __ballot(incl > t);
        if (past == 0) return false;
        const int first = __builtin_ctzll(past);
        int rest = t - (incl - mine), ee = -1, rr = 0, nn = 0;
        each([&](int x, int lo, int n) {
            const int c = large ? big(n) : small(n);
            if (rest >= 0 && rest < c) {
                const int skip = (large ? rest : n >> lg) << lg;
                ee = x, rr = lo + skip, nn = min(n - skip, 1 << lg);
            }
            rest -= c;
        });
        e = __builtin_amdgcn_readlane(ee, first);
        r0 = __builtin_amdgcn_readlane(rr, first);
        nr = __builtin_amdgcn_readlane(nn, first);
        return e >= 0 && nr > 0;
    }
};

// The item of workgroup `id` among `total`: workgroups go round-robin to the 8 XCDs (id % 8), and
// each XCD takes a contiguous run of items, so that neighbours share its L2. -1: none left.
__device__ __forceinline__ long xcd_item(long id, long total) {
    const long q = total / 8, rem = total % 8, x = id % 8, i = id / 8;
    if (i >= q + (x < rem)) return -1;
    return x * q + min(x, rem) + i;
}

// This workgroup's (tile, block of columns), columns fastest; false if it has none. The large
// tiles of all experts come before the small ones, each class spread evenly over the XCDs: 16384
// rows of 16 experts (four large tiles each, half of them with a few rows more) take two rounds of
// large items and a short one instead of three, 485 -> 410 us.
// halves: where the small items are at most kFewItems, which leaves half the CUs idle, they come in
// two halves of the columns, col counting halves (the same case 410 -> 387 us); 1 then, 0 for whole
// items.
constexpr int kFewItems = 128;
__device__ __forceinline__ bool find_item(const GroupedArgs& a, int lg, int& e, int& r0, int& nr,
                                          int& col, int* halves = nullptr) {
    const TileScan scan(a, lg);
    long id = blockIdx.x;
    const long big = (long)__builtin_amdgcn_readlane(scan.ibig, 63) * a.ntn;
    const long small = (long)__builtin_amdgcn_readlane(scan.ismall, 63) * a.ntn;
    const bool large = id < (big + 7) / 8 * 8;
    if (!large) id -= (big + 7) / 8 * 8;
    const int split = halves && !large && small <= kFewItems ? 1 : 0;
    if (halves) *halves = split;
    const long item = xcd_item(id, large ? big : small << split);
    if (item < 0) return false;
    const int ntn = a.ntn << split;
    long t = item / ntn;
    col = (int)(item % ntn);
    if (large && a.fours) {
        // Four tiles at a time: the 32 workgroups that an XCD runs together are 4 x 8 items and read
        // 12 operands' rows, not 33 (8192^3: 900 -> 854 us).
        const long nb = big / a.ntn, first = t / 4 * 4, rows = min(4L, nb - first);
        const long i = item - first * ntn;
        t = first + i % rows;
        col = (int)(i / rows);
    }
    return scan.find(large, (int)t, e, r0, nr);
}
// Workgroups for tiles of `rows` rows: as many as there may be tiles, and what the classes'
// rounding to 8 and the halves add.
static long grid_items(const GroupedArgs& a, int tile_rows) {
    const long groups = a.E + (a.sh_rows > 0), rows = (long)a.rows + a.sh_rows;
    return (rows / tile_rows + (groups < rows ? groups : rows)) * a.ntn + 16 + kFewItems;
}

// Tiles of rows x TN rows of W (TN / 2 features of both matrices where DUAL), 64 of K per
// step, D steps in LDS.
//
// Waves stand WR along the rows x WC along W: wave (wr, wc) has MB 16-row blocks wr, wr + WR, ...
// of the tile (so that a tile of few rows keeps every wave busy) and NB blocks of 16 rows of W. A
// row of a step is 128 B in LDS, its 16-byte chunk c at slot c ^ (row / 2 % 8): the 16 rows that
// a fragment read touches at one chunk fall on 16 different groups of banks. Rows go straight
// from memory to LDS, 8 whole rows to an instruction (steps of 32 K, 64 B a row, streamed W at
// 5.6 instead of 6.3 TB/s). Fragments are read one phase (up to 16 products) ahead; the one
// barrier of a step stands before its last phase: behind it the next step is complete and this
// step's LDS is free for the step D later.
constexpr int kTileK = 64;
// NT: W is read without a place in L2, where no other tile wants it (64 tokens of 8 of 256 experts, gate and
// up 6144 -> 2048: 1837 -> 1680 us, 6.7 TB/s; but 8192 rows of one expert, 8192 -> 8192, 869 -> 919).
// AL: rows of x and W are 16-byte aligned. Where they are not they come through registers, D = 2: loads of
// step s + 2 are asked for behind the barrier of step s and go to LDS before the next one.
template <class T, bool DUAL, bool F32, int WR, int WC, int NB, int LDS, bool NT, bool AL = true>
struct TileRun {
    static constexpr int W = WR * WC, TN = WC * NB * 16;
    const GroupedArgs& a;
    char* lds;
    int e, r0, nr, col, lane, wv;

    template <int MB>
    __device__ __forceinline__ void run() {
        constexpr int NP = MB > 4 ? 2 : 1, MH = (MB + NP - 1) / NP, PH = 2 * NP;
        constexpr int NA = MB * WR * 2, CA = (NA + W - 1) / W, CB = TN / 8 / W, BOFF = NA * 1024,
                      STAGE = (NA + TN / 8) * 1024, D0 = LDS / STAGE, D = !AL ? 2 : D0 < 8 ? D0 : 8;
        static_assert(D >= 2 && CB * W * 8 == TN, "two steps, whole instructions");
        const int r = lane & 15, q = lane >> 4, wr = wv / WC, wc = wv % WC;
        const int K = a.K, steps = (K + kTileK - 1) / kTileK;
        const uint16_t *w0 = a.w0 + (long)e * a.w_stride, *w1 = a.w1 + (long)e * a.w_stride;
        if (e == a.E) w0 = a.s0, w1 = a.s1;
        const int f0 = col * (DUAL ? TN / 2 : TN);

        // What this lane copies: chunk c8 of row lane / 8 of pieces of 8 rows. Of x, piece
        // W i + wv of the NA (waves past the last one repeat a piece).
        const int cr = lane >> 3;
        const uint16_t *pa[CA], *pb[CB];
        int at[CA], ka[CA], kb[CB];
        const uint32_t la = lds_addr(lds);
        // Chunks from K on are zeros (K % 8 == 0: a chunk is inside or not).
        auto fetch_w = [&](int s, uint32_t stage) {
            const int k = s * kTileK;
            const bool whole = k + kTileK <= K;
#pragma unroll
            for (int i = 0; i < CB; ++i)
                copy16<NT>(whole || k + kb[i] < K ? static_cast<const void*>(pb[i] + k) : &kZero16,
                       la + stage + BOFF + (W * i + wv) * 1024);
        };
        auto fetch_x = [&](int s, uint32_t stage) {
            const int k = s * kTileK;
            const bool whole = k + kTileK <= K;
#pragma unroll
            for (int i = 0; i < CA; ++i)
                copy16(whole || k + ka[i] < K ? static_cast<const void*>(pa[i] + k) : &kZero16,
                       la + stage + at[i] * 1024);
        };
        // The first steps' W is on its way while the rows of x are looked up.
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int j = 8 * (W * i + wv) + cr;    // row of W in the tile; a wave's are gate, then up
            const int n = DUAL ? f0 + j / (16 * NB) * 8 * NB + j % (8 * NB) : f0 + j;
            kb[i] = ((lane & 7) ^ (j >> 1 & 7)) * 8;
            pb[i] = (DUAL && j % (16 * NB) >= 8 * NB ? w1 : w0) + (long)min(n, a.N - 1) * K + kb[i];
        }
        int ids[CA];
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            at[i] = (W * i + wv) % NA;
            const int j = 8 * at[i] + cr, rr = j < nr ? r0 + j : r0;
            ids[i] = a.row_ids ? a.row_ids[rr] : rr;
            ka[i] = ((lane & 7) ^ (j >> 1 & 7)) * 8;
        }
        if constexpr (AL) {
#pragma unroll
            for (int s = 0; s < D - 1; ++s)
                if (s < steps) fetch_w(s, s * STAGE);
        }
#pragma unroll
        for (int i = 0; i < CA; ++i)
            pa[i] = a.x + (ids[i] >= 0 && ids[i] < a.x_rows ? (long)ids[i] : 0) * a.ldx + ka[i];
        if constexpr (AL) {
#pragma unroll
            for (int s = 0; s < D - 1; ++s)
                if (s < steps) fetch_x(s, s * STAGE);
        }
        auto fetch = [&](int s, uint32_t stage) {
            const int k = s * kTileK;
            if (k + kTileK <= K) {
#pragma unroll
                for (int i = 0; i < CB; ++i) copy16<NT>(pb[i] + k, la + stage + BOFF + (W * i + wv) * 1024);
#pragma unroll
                for (int i = 0; i < CA; ++i) copy16(pa[i] + k, la + stage + at[i] * 1024);
            } else {
                fetch_w(s, stage);
                fetch_x(s, stage);
            }
        };

        // Rows at any address: a step on its way in registers, cut at K when it goes to LDS.
        constexpr int CH = AL ? 1 : CA + CB;
        u32x4 held[CH];
        auto grab = [&](int s) __attribute__((always_inline)) {
            const int k = s * kTileK, top = K - 8;
#pragma unroll
            for (int i = 0; i < CH; ++i)
                held[i] = i < CB ? load8(pb[i] - kb[i], min(k + kb[i], top))
                                 : load8(pa[i - CB] - ka[i - CB], min(k + ka[i - CB], top));
        };
        auto drop = [&](int s, uint32_t stage) __attribute__((always_inline)) {
            const int k = s * kTileK;
            char* p = lds + stage + lane * 16;
            if (k + kTileK > K) {
#pragma unroll
                for (int i = 0; i < CH; ++i) held[i] = fit8(held[i], k + (i < CB ? kb[i] : ka[i - CB]), K);
            }
#pragma unroll
            for (int i = 0; i < CH; ++i)
                *reinterpret_cast<u32x4*>(p + (i < CB ? BOFF + (W * i + wv) * 1024 : at[i - CB] * 1024)) = held[i];
        };

        f32x4 acc[MB][NB];
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int n = 0; n < NB; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
        u32x4 fa[2][MH], fb[2][NB];
        // (Row / 2) % 8 is that of r in every block of 16 rows.
        const char* ra = lds + (wr * 16 + r) * 128;
        const char* rb = lds + BOFF + (wc * NB * 16 + r) * 128;
        const int c0 = (q ^ (r >> 1)) * 16;         // chunk q of half 0; half 1: chunk q + 4
        auto read = [&](uint32_t stage, int p) {    // phase p: half p / NP of K, rows p % NP
            const int kk = p / NP, h = p % NP, c = kk ? c0 ^ 64 : c0;
#pragma unroll
            for (int m = 0; m < MH; ++m)
                if (h * MH + m < MB)
                    fa[p & 1][m] = *reinterpret_cast<const u32x4*>(ra + stage + c + (h * MH + m) * WR * 2048);
            if (h == 0)
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    fb[kk][n] = *reinterpret_cast<const u32x4*>(rb + stage + c + n * 2048);
        };

        if constexpr (AL) {
            if (steps >= D - 1) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((D - 2) * CA) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("s_barrier" ::: "memory");
        } else {
            if (K >= 8) {
                grab(0);
            } else {            // one step, of rows too short for a load of eight
#pragma unroll
                for (int i = 0; i < CH; ++i)
                    held[i] = i < CB ? ask8(pb[i] - kb[i], 0, K) : ask8(pa[i - CB] - ka[i - CB], 0, K);
            }
            drop(0, 0);
            __syncthreads();
        }
        read(0, 0);
        if constexpr (AL) {
            if (D - 1 < steps) fetch(D - 1, (D - 1) * STAGE);
        } else {
            if (steps > 1) grab(1);
        }
        uint32_t cur = 0;
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int p = 0; p < PH; ++p) {
                if (p + 1 < PH) {
                    read(cur, p + 1);
                } else if (s + 1 < steps) {
                    // Step s + 1 has arrived, and this wave's reads of step s. What may be on its way then:
                    // D - 2 steps; before step D - 2, whose x was asked for after all the first W, less.
                    if constexpr (!AL) {
                        drop(s + 1, cur ^ STAGE);   // all have read step s - 1, which was there
                        __syncthreads();
                    } else if (s + D - 1 >= steps) {
                        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n s_barrier" ::: "memory");
                    } else if (s < D - 3) {
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n s_barrier" :: "n"((D - 2) * CA + CB) : "memory");
                    } else {
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n s_barrier" :: "n"((D - 2) * (CA + CB)) : "memory");
                    }
                    const uint32_t free = cur;
                    cur = cur + STAGE == D * STAGE ? 0 : cur + STAGE;
                    read(cur, 0);
                    if (s + D < steps) {
                        if constexpr (AL) fetch(s + D, free);
                        else grab(s + D);
                    }
                }
                const int kk = p / NP, h = p % NP;
#pragma unroll
                for (int m = 0; m < MH; ++m)
                    if (h * MH + m < MB)
#pragma unroll
                        for (int n = 0; n < NB; ++n)
                            acc[h * MH + m][n] = T::mma(fb[kk][n], fa[p & 1][m], acc[h * MH + m][n]);
            }
        }

        // A lane holds four neighbouring outputs of row `lane % 16` of each block.
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int j = (m * WR + wr) * 16 + r;
            if (j >= nr) continue;
            const int id = a.row_ids ? a.row_ids[r0 + j] : 0;
            const bool ok = !a.row_ids || (id >= 0 && id < a.x_rows);
            constexpr int NF = DUAL ? NB / 2 : NB;
#pragma unroll
            for (int n = 0; n < NF; ++n) {
                f32x4 v = acc[m][n];
                if constexpr (DUAL) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c] = silu_fast(v[c]) * acc[m][n + NF][c];
                }
                if (!ok) v = (f32x4){0.f, 0.f, 0.f, 0.f};
                const int f = f0 + (wc * NF + n) * 16 + 4 * q;
                if (f < a.N)
                    store4<T, F32>(a.y, (long)(r0 + j) * a.ldy + f, v, a.N - f);
            }
        }
    }
};

// Up to 256 rows x 256 rows of W, one workgroup of 8 waves to a CU.
template <class T, bool DUAL, bool F32, bool NT>
__global__ __launch_bounds__(512, 2) void grp_tile_kernel(GroupedArgs a) {
    __shared__ __align__(16) char lds[160 * 1024];
    TileRun<T, DUAL, F32, 2, 4, 4, 160 * 1024, NT> t{a, lds, 0, 0, 0, 0, (int)(threadIdx.x & 63),
                                                 __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
    int halves;
    if (!find_item(a, 8, t.e, t.r0, t.nr, t.col, &halves)) return;
    if (halves) {
        TileRun<T, DUAL, F32, 2, 4, 2, 160 * 1024, NT> h{a, lds, t.e, t.r0, t.nr, t.col, t.lane, t.wv};
        if (t.nr <= 32) h.template run<1>();
        else if (t.nr <= 64) h.template run<2>();
        else h.template run<4>();
    } else if (t.nr <= 32) t.template run<1>();
    else if (t.nr <= 64) t.template run<2>();
    else if (t.nr <= 128) t.template run<4>();
    else if (t.nr <= 160) t.template run<5>();
    else t.template run<8>();
}

// Up to 64 rows x 128 rows of W, two workgroups of 4 waves to a CU.
template <class T, bool DUAL, bool F32, bool NT>
__global__ __launch_bounds__(256, 2) void grp_slim_kernel(GroupedArgs a) {
    __shared__ __align__(16) char lds[80 * 1024];
    TileRun<T, DUAL, F32, 1, 4, 2, 80 * 1024, NT> t{a, lds, 0, 0, 0, 0, (int)(threadIdx.x & 63),
                                                __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
    if (!find_item(a, 6, t.e, t.r0, t.nr, t.col)) return;
    if (t.nr <= 16) t.template run<1>();
    else if (t.nr <= 32) t.template run<2>();
    else t.template run<4>();
}

// Rows at any address: up to 64 rows x 128 rows of W, three workgroups of 4 waves to a CU. What bounds it: 16-byte
// loads from odd multiples of 2 take 60 cycles of a CU's address unit for a wave, from multiples of 4 16
// (16384 rows of 16 experts, 2047 -> 2049: 337 us, 407 TFLOP/s); more steps on their way, and aligned
// loads whose two missing bytes come from the next lane, were no faster.
template <class T, bool DUAL, bool F32>
__global__ __launch_bounds__(256, 3) void grp_any_kernel(GroupedArgs a) {
    __shared__ __align__(16) char lds[48 * 1024];
    TileRun<T, DUAL, F32, 1, 4, 2, 48 * 1024, false, false> t{a, lds, 0, 0, 0, 0, (int)(threadIdx.x & 63),
                                                       __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
    if (!find_item(a, 6, t.e, t.r0, t.nr, t.col)) return;
    if (t.nr <= 16) t.template run<1>();
    else if (t.nr <= 32) t.template run<2>();
    else t.template run<4>();
}

// Rows per expert up to which the slim kernel runs: gate and up, 6144 -> 2048, 256 experts, at 16 / 32 / 64
// rows each 1.88 / 1.94 / 3.04 ms against the large kernel's 1.96 / 1.99 / 2.05; with 256 features and a skewed
// router (32 rows on average) 0.30 against 0.32.
constexpr int kSlimRows = 40;

// Rows per expert, on average over the experts that can have any.
static long mean_rows(const GroupedArgs& a) {
    const long rows = (long)a.rows + a.sh_rows, groups = a.E + (a.sh_rows > 0), g = groups < rows ? groups : rows;
    return (rows + g - 1) / g;
}

// Large tiles up to which the slim kernel runs, too: one workgroup of it has a CU to itself, and with less
// than two thirds of the CUs busy two smaller ones to each are faster (1332 rows of 13 experts, 1024 -> 515, 39
// tiles: 12 us against 35; 4096 rows of 8, 4096 -> 1792, 140: 86 against 107; 4096 rows of 64, 2048 ->
// 768, 192: 54 against 50).
constexpr int kFewTiles = 160;

template <class T, bool DUAL, bool F32>
static int run_tiles(const GroupedArgs& a0, bool aligned, hipStream_t s) {
    GroupedArgs a = a0;
    const long mean = mean_rows(a), rows = (long)a.rows + a.sh_rows, groups = a.E + (a.sh_rows > 0);
    const int wide = 256 / (DUAL ? 2 : 1);
    // An expert's last tile is half full on average, and it has one.
    const long g = groups < rows ? groups : rows, tiles = rows / 256 + g / 2;
    const bool few = mean <= kSlimRows,
               large = aligned && !few && (tiles > g ? tiles : g) * ((a.N + wide - 1) / wide) > kFewTiles;
    const int w = large ? wide : wide / 2;
    a.ntn = (a.N + w - 1) / w;
    // More rows: the tiles of an expert share its W. Fewer: W is read once and keeps out of L2.
    a.fours = mean > 256;
    const long items = grid_items(a, large ? 256 : 64);
    if (items * 512 >= (1L << 32)) return -2;     // threads of a launch
    const dim3 grid((unsigned)items);
    if (large && a.fours) hipLaunchKernelGGL((grp_tile_kernel<T, DUAL, F32, false>), grid, dim3(512), 0, s, a);
    else if (large) hipLaunchKernelGGL((grp_tile_kernel<T, DUAL, F32, true>), grid, dim3(512), 0, s, a);
    else if (!aligned) hipLaunchKernelGGL((grp_any_kernel<T, DUAL, F32>), grid, dim3(256), 0, s, a);
    else if (few) hipLaunchKernelGGL((grp_slim_kernel<T, DUAL, F32, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((grp_slim_kernel<T, DUAL, F32, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

// out[t] = sum over the slots s, in order, of w[t, s] * part[inv[t, s]], then the shared
// expert's row n topk + t: four features per thread, all rows loaded before the adds. A
// slot whose id is out of range has no row and counts nothing.
__global__ __launch_bounds__(256) void grp_combine_kernel(const float* __restrict__ part,
                                                          const int* __restrict__ inv,
                                                          const int* __restrict__ ids,
                                                          const float* __restrict__ w, int n,
                                                          int topk, int E, int H, int shared,
                                                          float* __restrict__ out) {
    const int nb = (H / 4 + 255) / 256;
    const int t = blockIdx.x / nb, f4 = blockIdx.x % nb * 256 + threadIdx.x;
    if (4 * f4 >= H) return;
    auto row = [&](long r) { return reinterpret_cast<const f32x4*>(part + r * H)[f4]; };
    f32x4 v[9];
    float ws[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        v[s] = (f32x4){0.f, 0.f, 0.f, 0.f};
        ws[s] = 0.0f;
        if (s < topk) {
            const long i = (long)t * topk + s;
            if (ids[i] >= 0 && ids[i] < E) {
                ws[s] = w[i];
                v[s] = row(inv[i]);
            }
        }
    }
    v[8] = shared ? row((long)n * topk + t) : (f32x4){0.f, 0.f, 0.f, 0.f};
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 8; ++s) acc += ws[s] * v[s];
    acc += v[8];
    reinterpret_cast<f32x4*>(out + (long)t * H)[f4] = acc;
}

int launch_grouped_combine(const float* part, const int* inv, const int* ids, const float* w, int n,
                           int topk, int E, int H, int shared, float* out, hipStream_t s) {
    const long grid = (long)n * ((H / 4 + 255) / 256);
    if (H % 4 || topk > 8 || grid * 256 >= (1L << 32)) return -2;
    hipLaunchKernelGGL(grp_combine_kernel, dim3((unsigned)grid), dim3(256), 0, s, part, inv, ids, w,
                       n, topk, E, H, shared, out);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <class T, bool DUAL>
static int run_types(const GroupedArgs& a, bool f32, hipStream_t s) {
    auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool aligned = a.K % 8 == 0 && a.ldx % 8 == 0 && a.w_stride % 8 == 0 && al(a.x) &&
                         al(a.w0) && (!DUAL || al(a.w1)) && al(a.s0) && al(a.s1);
    return f32 ? run_tiles<T, DUAL, true>(a, aligned, s) : run_tiles<T, DUAL, false>(a, aligned, s);
}

int launch_grouped(const GroupedArgs& a, int dtype, bool f32, hipStream_t s) {
    if (dtype == kBf16) return a.w1 ? run_types<Bf16, true>(a, f32, s) : run_types<Bf16, false>(a, f32, s);
    return a.w1 ? run_types<F16, true>(a, f32, s) : run_types<F16, false>(a, f32, s);
}

}  // namespace glmmoe
