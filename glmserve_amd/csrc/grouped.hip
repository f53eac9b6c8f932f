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

// Row tile t (tiles of 2^lg rows, in expert order) of the groups off[0 .. E]:
// its expert, first row and rows; false if there are fewer tiles. Every wave
// calls it and gets the same answer. Offsets are clamped to [0, rows], so that no
// tile leaves the rows whatever they hold.
__device__ __forceinline__ bool find_tile(const int* __restrict__ off, int E, int rows, int lg,
                                          int t, int& e, int& r0, int& nr) {
    const int lane = threadIdx.x & 63;
    const int per = (E + 63) / 64;
    auto at = [&](int i) { return min(max(off[min(i, E)], 0), rows); };
    auto tiles = [&](int i) { return i < E ? (max(at(i + 1) - at(i), 0) + (1 << lg) - 1) >> lg : 0; };
    int sum = 0;
    for (int j = 0; j < per; ++j) sum += tiles(lane * per + j);
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d);
        if (lane >= d) incl += v;
    }
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
    int e, r0, nr;
    const int tile = (int)(blockIdx.x / a.ntn);
    if (a.off) {
        if (!find_tile(a.off, a.E, a.rows, LG, tile, e, r0, nr)) return;
    } else {
        if (tile >= a.ntiles[0]) return;
        e = a.tiles[4 * tile], r0 = a.tiles[4 * tile + 1], nr = a.tiles[4 * tile + 2];
    }
    const uint16_t *w0 = a.w0 + (long)e * a.w_stride, *w1 = a.w1 + (long)e * a.w_stride;
    if (e == a.E) w0 = a.s0, w1 = a.s1;
    const int n0 = (int)(blockIdx.x % a.ntn) * 16 * NB;
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

int grouped_tile_rows(long rows, int E) {
    const long groups = E < rows ? E : rows;
    const long mean = (rows + groups - 1) / groups;
    return mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
}

template <class T, bool DUAL, bool AL, bool F32>
static int run_stream(const GroupedArgs& a0, hipStream_t s) {
    GroupedArgs a = a0;
    const int tb = a.off ? grouped_tile_rows(a.rows, a.E) / 16 : a.tb;
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
