// Low-rank adapters of many requests beside a shared projection:
//
//   y[t, :] = base[t, :] + scale[a] * B[a] (A[a] x[t]),   a = ids[t]
//
// in two launches: A x into fp32 partial sums (split over K, in order), then
// base + B (A x). No counterpart in the reference, whose linears (cuda/kernels.cuh:
// 37-66) this stands beside.
//
// Tokens keep their places: a workgroup takes a block of consecutive tokens and
// walks the adapters that occur in it, each once, with the tokens of the others
// computed along and dropped. Requests' tokens are neighbours in a batch, so a block
// of a prompt has one adapter, and decoding tokens with an adapter each need
// each adapter's weights once anyway.
#include "grouped.hpp"

#include "num16.hpp"

namespace glmmoe {

constexpr int kLoraWaves = 4;
constexpr int kRankBlocks = 4;            // ranks per workgroup of the first launch: 64

// 16-bit x fp32 products on the matrix cores: an fp32 value is the sum of three bf16
// terms of 8 bits each (truncation: exact; a value below 2^-110 loses its last bits, its
// terms being subnormal), an fp16 value of two.
struct Terms3 {
    u32x4 t[3];
};
__device__ __forceinline__ uint32_t hi16(uint32_t a, uint32_t b) {   // the upper halves of a (low), b
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
__device__ __forceinline__ void split3(float f, uint32_t& h, uint32_t& m, uint32_t& l) {
    const uint32_t u = __float_as_uint(f);
    const bool special = (u & 0x7f800000u) == 0x7f800000u;   // Inf, NaN: one term
    h = u | ((special && (u & 0x007fffffu)) ? 0x00400000u : 0u);
    const float r1 = f - __uint_as_float(u & 0xffff0000u);
    m = special ? 0u : __float_as_uint(r1);
    const float r2 = r1 - __uint_as_float(m & 0xffff0000u);
    l = special ? 0u : __float_as_uint(r2);
}
__device__ __forceinline__ Terms3 split3(const float (&f)[8]) {
    Terms3 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h0, m0, l0, h1, m1, l1;
        split3(f[2 * i], h0, m0, l0);
        split3(f[2 * i + 1], h1, m1, l1);
        o.t[0][i] = hi16(h0, h1);
        o.t[1][i] = hi16(m0, m1);
        o.t[2][i] = hi16(l0, l1);
    }
    return o;
}
// fp16 -> two bf16 terms.
__device__ __forceinline__ void split2(u32x4 v, u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[2], l[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float f = F16::up(v[i] >> (16 * c));
            const uint32_t u = __float_as_uint(f);
            h[c] = u;
            l[c] = (u & 0x7f800000u) == 0x7f800000u
                       ? 0u : __float_as_uint(f - __uint_as_float(u & 0xffff0000u));
        }
        hi[i] = hi16(h[0], h[1]);
        lo[i] = hi16(l[0], l[1]);
    }
}
// c += w * (t0 + t1 + t2), smallest terms first.
template <class W>
__device__ __forceinline__ f32x4 mma3(u32x4 w, const Terms3& t, f32x4 c) {
    if constexpr (W::code == kF16) {
        u32x4 hi, lo;
        split2(w, hi, lo);
#pragma unroll
        for (int i = 2; i >= 0; --i) c = Bf16::mma(lo, t.t[i], c);
        w = hi;
    }
#pragma unroll
    for (int i = 2; i >= 0; --i) c = Bf16::mma(w, t.t[i], c);
    return c;
}

// Eight values of a row of x as products take them.
template <class W>
struct XHalf {          // x of the adapters' type
    typedef uint16_t row_t;
    typedef u32x4 frag;
    template <bool AL>
    static __device__ __forceinline__ frag load(const row_t* p, int k) { return load8<AL>(p, k); }
    template <bool AL>
    static __device__ __forceinline__ frag tail(const row_t* p, int k, int K) { return load8_tail<AL>(p, k, K); }
    static __device__ __forceinline__ f32x4 mma(u32x4 w, const frag& x, f32x4 c) { return W::mma(w, x, c); }
};
template <class W>
struct XFloat {         // x fp32
    typedef float row_t;
    struct frag {
        float v[8];
    };
    template <bool AL>
    static __device__ __forceinline__ frag load(const row_t* p, int k) {
        frag f;
        if constexpr (AL) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + k), b = *reinterpret_cast<const f32x4*>(p + k + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { f.v[i] = a[i]; f.v[4 + i] = b[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f.v[i] = p[k + i];
        }
        return f;
    }
    template <bool AL>
    static __device__ __forceinline__ frag tail(const row_t* p, int k, int K) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f.v[i] = k + i < K ? p[k + i] : 0.0f;
        return f;
    }
    static __device__ __forceinline__ f32x4 mma(u32x4 w, const frag& x, f32x4 c) {
        return mma3<W>(w, split3(x.v), c);
    }
};

// The adapters of a block of tokens, one after the other: f(adapter, tokens as a mask of
// lanes) for every jn-th from j on. id: lane i's token's adapter, -1 for none.
template <class F>
__device__ __forceinline__ void each_adapter(int id, int j, int jn, F&& f) {
    uint64_t rest = __ballot(id >= 0);
    for (int i = 0; rest; ++i) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
        const uint64_t m = __ballot(id == a);
        rest &= ~m;
        if (i % jn == j) f(a, m);
    }
}
__device__ __forceinline__ int block_id(const LoraArgs& a, int t0, int tokens) {
    const int lane = threadIdx.x & 63, t = t0 + lane;
    const int id = lane < tokens && t < a.n ? a.ids[t] : -1;
    return id >= 0 && id < a.L ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs& a, int ad) {
    return a.ranks ? min(max(a.ranks[ad], 0), a.r) : a.r;
}

// part[split][t][:] = A[ids[t]][:, K of the split] x[t][K of the split]. A workgroup:
// 16 TB tokens, 64 ranks, one split; its waves take chunks of 32 KS of K in turn.
// A is the MFMA's A operand (D row = rank), x its B (D column = token).
template <class W, class X, int RB, int TB, bool AL>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_down_kernel(LoraArgs a) {
    constexpr int KS = 2, KC = 32 * KS;
    __shared__ f32x4 red[kLoraWaves][RB * TB][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    int id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int rg = a.rp / 16 > RB ? (a.rp / 16 + RB - 1) / RB : 1;
    const int rank0 = id % rg * RB * 16;
    id /= rg;
    const int j = id % a.jn, t0 = id / a.jn * 16 * TB;
    const int kb = split * a.kstep, ke = min(a.K, kb + a.kstep);
    const typename X::row_t* xp[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int tok = t0 + 16 * t + r;
        xp[t] = static_cast<const typename X::row_t*>(a.x) + (long)(tok < a.n ? tok : t0) * a.ldx;
    }
    each_adapter(block_id(a, t0, 16 * TB), j, a.jn, [&](int ad, uint64_t m) {
        const int rk = rank_of(a, ad);
        const int live = min((rk - rank0 + 15) / 16, RB);     // rank blocks with a rank in use
        f32x4 acc[RB][TB];
        const uint16_t* wp[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            wp[b] = a.A + ((long)ad * a.r + max(min(rank0 + 16 * b + r, rk - 1), 0)) * a.K;
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[b][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        if (live > 0) {
            int k = kb + wv * KC;
            for (; k + KC <= ke; k += KC * kLoraWaves) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 w[RB];
                    typename X::frag x[TB];
#pragma unroll
                    for (int b = 0; b < RB; ++b) w[b] = load8<AL>(wp[b], k + 32 * s + 8 * q);
#pragma unroll
                    for (int t = 0; t < TB; ++t) x[t] = X::template load<AL>(xp[t], k + 32 * s + 8 * q);
#pragma unroll
                    for (int b = 0; b < RB; ++b)
#pragma unroll
                        for (int t = 0; t < TB; ++t) acc[b][t] = X::mma(w[b], x[t], acc[b][t]);
                }
            }
            if (k < ke) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int kk = k + 32 * s + 8 * q;
                    typename X::frag x[TB];
#pragma unroll
                    for (int t = 0; t < TB; ++t) x[t] = X::template tail<AL>(xp[t], kk, ke);
#pragma unroll
                    for (int b = 0; b < RB; ++b) {
                        const u32x4 w = load8_tail<AL>(wp[b], kk, ke);
#pragma unroll
                        for (int t = 0; t < TB; ++t) acc[b][t] = X::mma(w, x[t], acc[b][t]);
                    }
                }
            }
        }
        __syncthreads();       // the last adapter's sums are read
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int t = 0; t < TB; ++t) red[wv][b * TB + t][lane] = acc[b][t];
        __syncthreads();
        for (int f = wv; f < RB * TB; f += kLoraWaves) {
            const int b = f / TB, t = f % TB, row = rank0 + 16 * b + 4 * q, tok = t0 + 16 * t + r;
            f32x4 v = red[0][f][lane];
#pragma unroll
            for (int w = 1; w < kLoraWaves; ++w) v += red[w][f][lane];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = row + c < rk ? v[c] : 0.0f;
            if (row < a.rp && (m >> (16 * t + r) & 1))
                *reinterpret_cast<f32x4*>(a.part + ((long)split * a.n + tok) * a.rp + row) = v;
        }
    });
}

// Four values of a row of base / y as fp32.
template <int DT>
__device__ __forceinline__ f32x4 get4(const void* p, long at, int cnt, bool vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DT == kF32) {
        const float* f = static_cast<const float*>(p) + at;
        if (vec) return *reinterpret_cast<const f32x4*>(f);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < cnt) v[i] = f[i];
    } else {
        const uint16_t* h = static_cast<const uint16_t*>(p) + at;
        u32x2 w = {0u, 0u};
        if (vec) {
            w = *reinterpret_cast<const u32x2*>(h);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < cnt) w[i / 2] |= (uint32_t)h[i] << (16 * (i & 1));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = w[i / 2] >> (16 * (i & 1));
            v[i] = DT == kBf16 ? Bf16::up(u) : F16::up(u);
        }
    }
    return v;
}
template <int DT>
__device__ __forceinline__ void put4(void* p, long at, f32x4 v, int cnt, bool vec) {
    if constexpr (DT == kF16) store4<F16, false>(p, at, v, cnt, vec);
    else store4<Bf16, DT == kF32>(p, at, v, cnt, vec);
}

// y = base + scale * B (sum of part over the splits). A workgroup: 16 TB tokens, 256
// columns, 64 per wave; A x is summed, cut into three bf16 terms and kept in LDS.
// B is the MFMA's A operand (D row = output), A x its B (D column = token): a lane has
// four neighbouring outputs of one token.
template <class W, int YD, int TB, bool AL>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_up_kernel(LoraArgs a) {
    constexpr int NB = 4;
    extern __shared__ uint16_t terms[];              // [3][16 TB][stride]
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int stride = (a.r + 31) / 32 * 32 + 8;
    int id = blockIdx.x;
    const int n0 = (id % a.nx * kLoraWaves + wv) * 16 * NB;
    id /= a.nx;
    const int j = id % a.jn, t0 = id / a.jn * 16 * TB;
    const int ad0 = block_id(a, t0, 16 * TB);
    const uint64_t has = __ballot(ad0 >= 0);
    auto word = [&](int term, int t, int k) { return terms + ((term * 16 * TB + t) * stride + k); };

    for (int i = threadIdx.x; i < 16 * TB * (stride / 8); i += 64 * kLoraWaves) {
        const int t = i / (stride / 8), k = i % (stride / 8) * 8;
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = 0.0f;
        if (k < a.rp && (has >> t & 1)) {
            for (int s = 0; s < a.splits; ++s) {
                const float* p = a.part + ((long)s * a.n + t0 + t) * a.rp + k;
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] += p[c];
            }
        }
        const Terms3 o = split3(v);
#pragma unroll
        for (int c = 0; c < 3; ++c) *reinterpret_cast<u32x4*>(word(c, t, k)) = o.t[c];
    }
    __syncthreads();

    auto each_out = [&](uint64_t m, auto&& value) {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int tok = t0 + 16 * t + r;
            if (!(m >> (16 * t + r) & 1)) continue;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int n = n0 + 16 * b + 4 * q;
                if (n >= a.N) continue;
                const bool vec = a.vec && n + 4 <= a.N;
                const f32x4 v = get4<YD>(a.base, (long)tok * a.ldb + n, a.N - n, vec);
                put4<YD>(a.y, (long)tok * a.ldy + n, value(b, t, v), a.N - n, vec);
            }
        }
    };
    if (j == 0 && a.y != a.base) {                    // tokens without an adapter
        const int left = a.n - t0;
        const uint64_t here = left >= 64 ? ~0ull : (1ull << left) - 1;
        const uint64_t none = ~has & here & (TB == 4 ? ~0ull : (1ull << (16 * TB)) - 1);
        each_out(none, [](int, int, f32x4 v) { return v; });
    }
    each_adapter(ad0, j, a.jn, [&](int ad, uint64_t m) {
        const int rk = rank_of(a, ad);
        const float sc = a.scale ? a.scale[ad] : 1.0f;
        f32x4 acc[NB][TB];
        const uint16_t* wp[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            wp[b] = a.B + ((long)ad * a.N + min(n0 + 16 * b + r, a.N - 1)) * a.r;
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[b][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        for (int k = 0; k < rk; k += 32) {
            const int kk = k + 8 * q;
            Terms3 x[TB];
#pragma unroll
            for (int t = 0; t < TB; ++t)
#pragma unroll
                for (int c = 0; c < 3; ++c) x[t].t[c] = *reinterpret_cast<const u32x4*>(word(c, 16 * t + r, kk));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const u32x4 w = load8_tail<false>(wp[b], kk, rk);
#pragma unroll
                for (int t = 0; t < TB; ++t) acc[b][t] = mma3<W>(w, x[t], acc[b][t]);
            }
        }
        each_out(m, [&](int b, int t, f32x4 v) {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = __builtin_fmaf(sc, acc[b][t][c], v[c]);
            return v;
        });
    });
}

// How the first launch splits K: enough workgroups to fill the chip, 256 of K at least.
struct LoraPlan {
    int tb, blocks, jn, splits, kstep, rp;
};
static LoraPlan plan_of(int n, int L, int K, int r) {
    LoraPlan p;
    p.tb = n > 1024 ? 2 : 1;
    p.blocks = (n + 16 * p.tb - 1) / (16 * p.tb);
    const int most = n < L ? n : L;
    p.jn = n > 512 ? 1 : most < 16 ? most : 16;
    p.rp = (r + 15) / 16 * 16;
    const long wgs = (long)p.blocks * p.jn * ((r + 16 * kRankBlocks - 1) / (16 * kRankBlocks));
    long s = (512 + wgs - 1) / wgs;
    const int top = (K + 255) / 256;
    s = s < 1 ? 1 : s > top ? top : s;
    p.kstep = (int)(((K + s - 1) / s + 127) / 128 * 128);
    p.splits = (K + p.kstep - 1) / p.kstep;
    return p;
}
size_t lora_part_bytes(int n, int L, int K, int r) {
    const LoraPlan p = plan_of(n, L, K, r);
    return (size_t)p.splits * n * p.rp * 4;
}

template <class W, class X, bool AL>
static void run_down(const LoraArgs& a, const LoraPlan& p, unsigned grid, hipStream_t s) {
    const dim3 g(grid), b(64 * kLoraWaves);
    const int rb = p.rp / 16;
    auto go = [&](auto tb) {
        constexpr int TB = decltype(tb)::value;
        if (rb == 1) hipLaunchKernelGGL((lora_down_kernel<W, X, 1, TB, AL>), g, b, 0, s, a);
        else if (rb == 2) hipLaunchKernelGGL((lora_down_kernel<W, X, 2, TB, AL>), g, b, 0, s, a);
        else hipLaunchKernelGGL((lora_down_kernel<W, X, 4, TB, AL>), g, b, 0, s, a);
    };
    if (p.tb == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
}

template <class W, int YD>
static int run_up(const LoraArgs& a0, hipStream_t s) {
    LoraArgs a = a0;
    const int tb = a.n > 1024 && a.r <= 128 ? 4 : 1;   // 52 KiB of LDS at most
    const long blocks = (a.n + 16 * tb - 1) / (16 * tb);
    a.nx = (a.N + 255) / 256;
    if (tb == 4) a.jn = 1;
    const long grid = blocks * a.jn * a.nx;
    if (grid >= (1L << 31)) return -2;
    const size_t lds = (size_t)3 * 16 * tb * ((a.r + 31) / 32 * 32 + 8) * 2;
    const dim3 g((unsigned)grid), b(64 * kLoraWaves);
    if (tb == 1) hipLaunchKernelGGL((lora_up_kernel<W, YD, 1, true>), g, b, lds, s, a);
    else hipLaunchKernelGGL((lora_up_kernel<W, YD, 4, true>), g, b, lds, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int launch_lora(const LoraArgs& a0, int xdt, int wdt, int ydt, hipStream_t s) {
    LoraArgs a = a0;
    const LoraPlan p = plan_of(a.n, a.L, a.K, a.r);
    a.splits = p.splits, a.kstep = p.kstep, a.rp = p.rp, a.jn = p.jn;
    auto al = [](const void* q, size_t v) { return reinterpret_cast<uintptr_t>(q) % v == 0; };
    const size_t yb = ydt == kF32 ? 16 : 8;
    a.vec = a.ldb % 4 == 0 && a.ldy % 4 == 0 && al(a.base, yb) && al(a.y, yb);
    const bool aligned = a.K % 8 == 0 && al(a.x, 16) && al(a.A, 16) && a.ldx % (xdt == kF32 ? 4 : 8) == 0;
    const long grid = (long)p.blocks * p.jn * ((p.rp / 16 + kRankBlocks - 1) / kRankBlocks) * p.splits;
    if (grid >= (1L << 31)) return -2;
    auto down = [&](auto w) {
        using W = decltype(w);
        const unsigned g = (unsigned)grid;
        if (xdt == kF32) aligned ? run_down<W, XFloat<W>, true>(a, p, g, s) : run_down<W, XFloat<W>, false>(a, p, g, s);
        else aligned ? run_down<W, XHalf<W>, true>(a, p, g, s) : run_down<W, XHalf<W>, false>(a, p, g, s);
    };
    if (wdt == kBf16) down(Bf16{});
    else down(F16{});
    if (hipGetLastError() != hipSuccess) return -4;
    if (wdt == kBf16) return ydt == kF32 ? run_up<Bf16, kF32>(a, s) : run_up<Bf16, kBf16>(a, s);
    return ydt == kF32 ? run_up<F16, kF32>(a, s) : run_up<F16, kF16>(a, s);
}

}  // namespace glmmoe
