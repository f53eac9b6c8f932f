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

// Row tiles (2^lg rows at most, in expert order) of the groups off[0 .. E]: how many, and the
// expert, first row and rows of one. Every wave calls it and gets the same answer. Offsets
// are clamped to [0, rows], so that no tile leaves the rows whatever they hold.
struct TileScan {
    const int* off;
    int E, rows, lg, per, sum, incl;

    __device__ __forceinline__ int at(int i) const { return min(max(off[min(i, E)], 0), rows); }
    __device__ __forceinline__ int tiles(int i) const {
        return i < E ? (max(at(i + 1) - at(i), 0) + (1 << lg) - 1) >> lg : 0;
    }
    __device__ __forceinline__ TileScan(const int* o, int E_, int rows_, int lg_)
        : off(o), E(E_), rows(rows_), lg(lg_), per((E_ + 63) / 64), sum(0) {
        const int lane = threadIdx.x & 63;
        for (int j = 0; j < per; ++j) sum += tiles(lane * per + j);
        incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(incl, d);
            if (lane >= d) incl += v;
        }
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(incl, 63); }
    __device__ __forceinline__ bool find(int t, int& e, int& r0, int& nr) const {
        const uint64_t past = __ballot(incl > t);
        if (past == 0) return false;
        const int first = __builtin_ctzll(past);
        int rest = t - __builtin_amdgcn_readlane(incl - sum, first);
        e = first * per;
        for (int j = 1, c = tiles(e); j < per && rest >= c; ++j, c = tiles(++e)) rest -= c;
        e = __builtin_amdgcn_readfirstlane(e);
        rest = __builtin_amdgcn_readfirstlane(rest);
        r0 = __builtin_amdgcn_readfirstlane(at(e)) + (rest << lg);
        nr = min(__builtin_amdgcn_readfirstlane(at(e + 1)) - r0, 1 << lg);
        return e < E && nr > 0;
    }
};

// The item of workgroup `id` among `total`: workgroups go round-robin to the 8 XCDs (id % 8), and
// each XCD takes a contiguous run of items, so that neighbours share its L2. -1: none left.
__device__ __forceinline__ long xcd_item(long id, long total) {
    const long q = total / 8, rem = total % 8, x = id % 8, i = id / 8;
    if (i >= q + (x < rem)) return -1;
    return x * q + min(x, rem) + i;
}

// This workgroup's (tile, block of columns), columns fastest; false if it has none.
__device__ __forceinline__ bool find_item(const GroupedArgs& a, int lg, int& e, int& r0, int& nr,
                                          int& col) {
    if (a.off) {
        const TileScan scan(a.off, a.E, a.rows, lg);
        const long item = xcd_item(blockIdx.x, (long)scan.total() * a.ntn);
        if (item < 0) return false;
        col = (int)(item % a.ntn);
        return scan.find((int)(item / a.ntn), e, r0, nr);
    }
    const long item = xcd_item(blockIdx.x, (long)min(a.ntiles[0], a.max_tiles) * a.ntn);
    if (item < 0) return false;
    col = (int)(item % a.ntn);
    const int* t = a.tiles + 4 * (item / a.ntn);
    e = t[0], r0 = t[1], nr = t[2];
    return true;
}

// Few rows per expert: the weights are streamed once and bound the time.
// A workgroup has one tile of 16 TB rows and 16 NB rows of W (of each of the two
// matrices where DUAL) over all of K; its 4 waves take chunks of 32 KS of K in
// turn, straight from memory to registers, the next chunk's loads before this
// chunk's products, and add their sums in LDS in order. W is the MFMA's A operand
// (D row = output feature) and x its B (D column = row of the tile), so a lane
// stores four consecutive features of one row. Columns past the tile's rows repeat
// its first row and are dropped.
constexpr int kStreamWaves = 4;

template <class T, bool DUAL, int NB, int TB, int KS, bool AL, bool F32>
__global__ __launch_bounds__(64 * kStreamWaves) void grp_stream_kernel(GroupedArgs a) {
    constexpr int M = DUAL ? 2 : 1, LG = TB == 1 ? 4 : TB == 2 ? 5 : 6, KC = 32 * KS;
    __shared__ f32x4 red[kStreamWaves][M * NB * TB][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    int e, r0, nr, col;
    if (!find_item(a, LG, e, r0, nr, col)) return;
    const uint16_t *w0 = a.w0 + (long)e * a.w_stride, *w1 = a.w1 + (long)e * a.w_stride;
    if (e == a.E) w0 = a.s0, w1 = a.s1;
    const int n0 = col * 16 * NB;
    const int K = a.K;

    const uint16_t* xp[TB];
    bool ok[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int j = t * 16 + r, rr = j < nr ? r0 + j : r0;
        const int id = a.row_ids ? a.row_ids[rr] : rr;
        ok[t] = id >= 0 && id < a.x_rows;
        xp[t] = a.x + (ok[t] ? (long)id : 0) * a.ldx;
    }
    const uint16_t* wp[M][NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const long at = (long)min(n0 + 16 * b + r, a.N - 1) * K;
        wp[0][b] = w0 + at;
        if constexpr (DUAL) wp[1][b] = w1 + at;
    }

    f32x4 acc[M][NB][TB];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[m][b][t] = (f32x4){0.f, 0.f, 0.f, 0.f};

    struct Chunk {
        u32x4 w[M][NB][KS], x[TB][KS];
    };
    auto load = [&](Chunk& c, int k0) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int b = 0; b < NB; ++b) c.w[m][b][s] = load8<AL, AL>(wp[m][b], k0 + 32 * s + 8 * q);
#pragma unroll
            for (int t = 0; t < TB; ++t) c.x[t][s] = load8<AL>(xp[t], k0 + 32 * s + 8 * q);
        }
    };
    auto mul = [&](const Chunk& c) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int t = 0; t < TB; ++t)
                        acc[m][b][t] = T::mma(c.w[m][b][s], c.x[t][s], acc[m][b][t]);
    };
    constexpr int STEP = KC * kStreamWaves;
    const int full = K / KC;                       // whole chunks; wave w takes w, w + 4, ...
    int i = wv;
    if (i < full) {
        Chunk c0, c1;
        load(c0, i * KC);
        for (;;) {
            i += kStreamWaves;
            const bool more = i < full;
            if (more) load(c1, i * KC);
            mul(c0);
            if (!more) break;
            i += kStreamWaves;
            const bool more2 = i < full;
            if (more2) load(c0, i * KC);
            mul(c1);
            if (!more2) break;
        }
    }
    if (full * KC < K && full % kStreamWaves == wv) {   // the rest of K, zeros after it
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int k = full * KC + 32 * s + 8 * q;
            u32x4 x[TB];
#pragma unroll
            for (int t = 0; t < TB; ++t) x[t] = load8_tail<AL>(xp[t], k, K);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const u32x4 w = load8_tail<AL>(wp[m][b], k, K);
#pragma unroll
                    for (int t = 0; t < TB; ++t) acc[m][b][t] = T::mma(w, x[t], acc[m][b][t]);
                }
        }
    }

#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < TB; ++t) red[wv][(m * NB + b) * TB + t][lane] = acc[m][b][t];
    __syncthreads();
    auto total = [&](int f) {
        f32x4 v = red[0][f][lane];
#pragma unroll
        for (int w = 1; w < kStreamWaves; ++w) v += red[w][f][lane];
        return v;
    };
    for (int f = wv; f < NB * TB; f += kStreamWaves) {
        const int b = f / TB, t = f % TB, j = t * 16 + r, n = n0 + 16 * b + 4 * q;
        f32x4 v = total(f);
        if constexpr (DUAL) {
            const f32x4 u = total(NB * TB + f);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = silu_fast(v[c]) * u[c];
        }
        bool good = true;
#pragma unroll
        for (int c = 0; c < TB; ++c) good = c == t ? ok[c] : good;
        if (!good) v = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (j < nr && n < a.N)
            store4<T, F32>(a.y, (long)(r0 + j) * a.ldy + n, v, a.N - n, a.vec && n + 4 <= a.N);
    }
}

// Many rows per expert: tiles of up to 256 rows x 256 rows of W (128 features of both
// matrices where DUAL), 64 of K per step, two steps' operands in LDS.
//
// 8 waves, 2 along the rows x 4 along W: wave (wr, wc) has the 16-row blocks wr, wr + 2, ... of
// the tile (so that a tile of few rows keeps both wave rows busy) and 64 rows of W. A row of a
// step is 128 B in LDS, its 16-byte chunk c at slot c ^ (row / 2 % 8): the 16 rows that a
// fragment read touches at one chunk fall on 16 different groups of banks. Whole rows go
// straight from memory to LDS, 8 to an instruction. A step has two 32-K halves of one or two row halves
// each ("phases" of 16 MFMAs); the next phase's fragments are read before this phase's products,
// and the one barrier of a step stands before its last phase: behind it the next step is complete
// and the step's own half of LDS is free for the step after that.
constexpr int kTileWaves = 8, kTileN = 256, kTileK = 64;
constexpr int kTileHalf = 256 * 128;              // LDS bytes of one operand of a step
constexpr int kTileLds = 4 * kTileHalf;
__device__ const u32x4 grp_zero = {0u, 0u, 0u, 0u};

// 64 lanes x 16 B from memory to LDS at base + 16 * lane, without the compiler's knowledge: it
// would have every LDS read wait for all of them.
__device__ __forceinline__ void copy16(const void* g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n s_nop 0\n global_load_lds_dwordx4 %0, off"
                 :: "v"(g), "s"(lds) : "memory");
}

template <class T, bool DUAL, bool AL, bool F32>
struct TileRun {
    const GroupedArgs& a;
    char* lds;
    int e, r0, nr, col, lane, wv;

    // MB: 16-row blocks per wave row.
    template <int MB>
    __device__ __forceinline__ void run() {
        constexpr int MH = MB < 4 ? MB : 4, NP = MB / MH, PH = 2 * NP, CA = MB / 2;
        const int r = lane & 15, q = lane >> 4, wr = wv >> 2, wc = wv & 3;
        const int K = a.K, steps = (K + kTileK - 1) / kTileK;
        const uint16_t *w0 = a.w0 + (long)e * a.w_stride, *w1 = a.w1 + (long)e * a.w_stride;
        if (e == a.E) w0 = a.s0, w1 = a.s1;
        const int f0 = col * (DUAL ? kTileN / 2 : kTileN);

        // What this lane copies: chunk `c8` of rows (8 i + wv) * 8 + lane / 8.
        const int cr = wv * 8 + (lane >> 3), c8 = ((lane & 7) ^ (cr >> 1 & 7)) * 8;
        const uint16_t *pa[CA], *pb[4];
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            const int j = 64 * i + cr, rr = j < nr ? r0 + j : r0;
            const int id = a.row_ids ? a.row_ids[rr] : rr;
            pa[i] = a.x + (id >= 0 && id < a.x_rows ? (long)id : 0) * a.ldx;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 64 * i + cr;              // row of W in the tile: 64 to a wave column
            const int n = DUAL ? f0 + (j >> 6) * 32 + (j & 31) : f0 + j;
            pb[i] = (DUAL && (j & 32) ? w1 : w0) + (long)min(n, a.N - 1) * K;
        }
        const uint32_t la = lds_addr(lds);
        auto fetch = [&](int s) {
            const uint32_t at = la + (s & 1) * 2 * kTileHalf + wv * 1024;
            const int k = s * kTileK + c8;
            const bool in = k < K;                  // K % 8 == 0: a chunk is inside or not
#pragma unroll
            for (int i = 0; i < CA; ++i)
                copy16(in ? static_cast<const void*>(pa[i] + k) : &grp_zero, at + i * 8192);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                copy16(in ? static_cast<const void*>(pb[i] + k) : &grp_zero, at + kTileHalf + i * 8192);
        };
        auto frag = [&](int buf, int operand, int row, int kk) {
            const int c = (kk * 4 + q) ^ (row >> 1 & 7);
            return *reinterpret_cast<const u32x4*>(lds + buf * 2 * kTileHalf + operand * kTileHalf +
                                                   row * 128 + c * 16);
        };

        f32x4 acc[MB][4];
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
        u32x4 fa[2][MH], fb[2][4];
        auto read = [&](int buf, int p) {           // phase p: half p / NP of K, rows p % NP
            const int kk = p / NP, h = p % NP;
#pragma unroll
            for (int m = 0; m < MH; ++m)
                fa[p & 1][m] = frag(buf, 0, ((h * MH + m) * 2 + wr) * 16 + r, kk);
            if (h == 0)
#pragma unroll
                for (int n = 0; n < 4; ++n) fb[kk][n] = frag(buf, 1, wc * 64 + n * 16 + r, kk);
        };

        fetch(0);
        if (steps > 1) {
            fetch(1);
            asm volatile("s_waitcnt vmcnt(%0)" :: "n"(CA + 4) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        asm volatile("s_barrier" ::: "memory");
        read(0, 0);
        for (int s = 0; s < steps; ++s) {
            const int buf = s & 1;
#pragma unroll
            for (int p = 0; p < PH; ++p) {
                if (p + 1 < PH) {
                    read(buf, p + 1);
                } else if (s + 1 < steps) {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n s_barrier" ::: "memory");
                    read(buf ^ 1, 0);
                    if (s + 2 < steps) fetch(s + 2);
                }
                const int kk = p / NP, h = p % NP;
#pragma unroll
                for (int m = 0; m < MH; ++m)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        acc[h * MH + m][n] = T::mma(fb[kk][n], fa[p & 1][m], acc[h * MH + m][n]);
            }
        }

        // A lane holds four neighbouring outputs of row `lane % 16` of each block.
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int j = (m * 2 + wr) * 16 + r;
            if (j >= nr) continue;
            const int id = a.row_ids ? a.row_ids[r0 + j] : 0;
            const bool ok = !a.row_ids || (id >= 0 && id < a.x_rows);
#pragma unroll
            for (int n = 0; n < (DUAL ? 2 : 4); ++n) {
                f32x4 v = acc[m][n];
                if constexpr (DUAL) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c] = silu_fast(v[c]) * acc[m][n + 2][c];
                }
                if (!ok) v = (f32x4){0.f, 0.f, 0.f, 0.f};
                const int f = f0 + wc * (DUAL ? 32 : 64) + 16 * n + 4 * q;
                if (f < a.N)
                    store4<T, F32>(a.y, (long)(r0 + j) * a.ldy + f, v, a.N - f, a.vec && f + 4 <= a.N);
            }
        }
    }
};

template <class T, bool DUAL, bool AL, bool F32>
__global__ __launch_bounds__(64 * kTileWaves, 2) void grp_tile_kernel(GroupedArgs a) {
    __shared__ __align__(16) char lds[kTileLds];
    TileRun<T, DUAL, AL, F32> t{a, lds, 0, 0, 0, 0, (int)(threadIdx.x & 63),
                                __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
    if (!find_item(a, 8, t.e, t.r0, t.nr, t.col)) return;
    if (t.nr <= 64) t.template run<2>();
    else if (t.nr <= 128) t.template run<4>();
    else t.template run<8>();
}

int grouped_tile_rows(long rows, int E) {
    const long groups = E < rows ? E : rows;
    const long mean = (rows + groups - 1) / groups;
    return mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 48 ? 64 : 256;
}

template <class T, bool DUAL, bool AL, bool F32>
static int run_stream(const GroupedArgs& a0, hipStream_t s) {
    GroupedArgs a = a0;
    int tb = a.off ? grouped_tile_rows(a.rows, a.E) / 16 : a.tb;
    if (AL && tb == 16) {
        const int w = DUAL ? kTileN / 2 : kTileN;
        a.ntn = (a.N + w - 1) / w;
        const long items = (a.off ? (long)a.rows / 256 + (a.E < a.rows ? a.E : a.rows) : a.max_tiles) * a.ntn;
        if (items >= (1L << 31)) return -2;
        hipLaunchKernelGGL((grp_tile_kernel<T, DUAL, AL, F32>), dim3((unsigned)items),
                           dim3(64 * kTileWaves), 0, s, a);
        return hipGetLastError() == hipSuccess ? 0 : -4;
    }
    if (tb > 4) tb = 4;
    constexpr int NB = DUAL ? 1 : 2;
    a.ntn = (a.N + 16 * NB - 1) / (16 * NB);
    const long tiles = a.off ? (long)a.rows / (16 * tb) + (a.E < a.rows ? a.E : a.rows) : a.max_tiles;
    const long grid = tiles * a.ntn;
    if (grid >= (1L << 31)) return -2;
    const dim3 g((unsigned)grid), b(64 * kStreamWaves);
    if (tb == 1) hipLaunchKernelGGL((grp_stream_kernel<T, DUAL, NB, 1, 4, AL, F32>), g, b, 0, s, a);
    else if (tb == 2) hipLaunchKernelGGL((grp_stream_kernel<T, DUAL, NB, 2, 4, AL, F32>), g, b, 0, s, a);
    else hipLaunchKernelGGL((grp_stream_kernel<T, DUAL, NB, 4, 2, AL, F32>), g, b, 0, s, a);
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
    if (H % 4 || topk > 8 || grid >= (1L << 31)) return -2;
    hipLaunchKernelGGL(grp_combine_kernel, dim3((unsigned)grid), dim3(256), 0, s, part, inv, ids, w,
                       n, topk, E, H, shared, out);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <class T, bool DUAL>
static int run_types(const GroupedArgs& a, bool f32, hipStream_t s) {
    auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool aligned = a.K % 8 == 0 && a.ldx % 8 == 0 && a.w_stride % 8 == 0 && al(a.x) &&
                         al(a.w0) && (!DUAL || al(a.w1)) && al(a.s0) && al(a.s1);
    if (aligned) return f32 ? run_stream<T, DUAL, true, true>(a, s) : run_stream<T, DUAL, true, false>(a, s);
    return f32 ? run_stream<T, DUAL, false, true>(a, s) : run_stream<T, DUAL, false, false>(a, s);
}

int launch_grouped(const GroupedArgs& a0, int dtype, bool f32, hipStream_t s) {
    GroupedArgs a = a0;
    const uintptr_t ya = reinterpret_cast<uintptr_t>(a.y);
    a.vec = a.ldy % 4 == 0 && ya % (f32 ? 16 : 8) == 0;
    if (dtype == kBf16) return a.w1 ? run_types<Bf16, true>(a, f32, s) : run_types<Bf16, false>(a, f32, s);
    return a.w1 ? run_types<F16, true>(a, f32, s) : run_types<F16, false>(a, f32, s);
}

}  // namespace glmmoe
