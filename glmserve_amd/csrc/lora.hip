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
    static __device__ __forceinline__ frag load(const row_t* p, int k) { return load8(p, k); }
    static __device__ __forceinline__ frag tail(const row_t* p, int k, int K) { return load8_tail(p, k, K); }
    // Values 8 c .. 8 c + 7 of a step's row r at p.
    static __device__ __forceinline__ void lds(const char* p, int c, int r, frag& x) {
        x = *reinterpret_cast<const u32x4*>(p + (c ^ r) * 16);
    }
    static __device__ __forceinline__ u32x4 split(const frag& x) { return x; }
    static __device__ __forceinline__ f32x4 mma(u32x4 w, u32x4 x, f32x4 c) { return W::mma(w, x, c); }
};
template <class W>
struct XFloat {         // x fp32
    typedef float row_t;
    struct frag {
        float v[8];
    };
    static __device__ __forceinline__ frag of(f32x4 a, f32x4 b) {
        frag f;
#pragma unroll
        for (int i = 0; i < 4; ++i) { f.v[i] = a[i]; f.v[4 + i] = b[i]; }
        return f;
    }
    static __device__ __forceinline__ frag load(const row_t* p, int k) {
        return of(*reinterpret_cast<const f32x4_any*>(p + k), *reinterpret_cast<const f32x4_any*>(p + k + 4));
    }
    static __device__ __forceinline__ frag tail(const row_t* p, int k, int K) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f.v[i] = k + i < K ? p[k + i] : 0.0f;
        return f;
    }
    static __device__ __forceinline__ void lds(const char* p, int c, int r, frag& x) {
        x = of(*reinterpret_cast<const f32x4*>(p + ((2 * c) ^ r) * 16),
               *reinterpret_cast<const f32x4*>(p + ((2 * c + 1) ^ r) * 16));
    }
    static __device__ __forceinline__ Terms3 split(const frag& x) { return split3(x.v); }
    static __device__ __forceinline__ f32x4 mma(u32x4 w, const Terms3& x, f32x4 c) { return mma3<W>(w, x, c); }
};

// What a workgroup does of the tokens' blocks (16 TB tokens each): the j-th adapter of a block and every
// jn-th after it. The workgroups that few blocks need come first, so that those that all blocks need
// fill all XCDs (id % 8) evenly: a batch of prompts has one adapter in a block, but where its decoding
// requests stand, before or after them, a block has many, so the blocks of the first and last
// 64 tokens have je workgroups, the others jm. Blocks go from the last to the first.
constexpr int kEndTokens = 64;
template <int TB>
struct BlockItem {
    int t0, j, jn;
    static __host__ __device__ __forceinline__ int blocks(int n) { return (n + 16 * TB - 1) / (16 * TB); }
    static __host__ __device__ __forceinline__ int ends(int n) {
        const int both = 2 * kEndTokens / (16 * TB), b = blocks(n);
        return b < both ? b : both;
    }
    static __host__ __forceinline__ long count(const LoraArgs& a) {
        return (long)blocks(a.n) * a.jm + (long)ends(a.n) * (a.je - a.jm);
    }
    __device__ __forceinline__ BlockItem(const LoraArgs& a, int id) {
        constexpr int EB = kEndTokens / (16 * TB);
        const int nb = blocks(a.n), ne = ends(a.n), more = a.je - a.jm;
        int b;
        if (id < ne * more) {
            const int e = id / more;
            b = e < EB ? e : nb - ne + e;
            j = a.jm + id % more;
        } else {
            id -= ne * more;
            b = nb - 1 - id % nb;
            j = a.jm - 1 - id / nb;
        }
        t0 = b * 16 * TB;
        jn = b < EB || b >= nb - (ne - EB) ? a.je : a.jm;
    }
};

// The adapters of a block of tokens, one after the other, every jn-th from the j-th on.
struct Adapters {
    int id;                   // lane i: its token's adapter, -1 for none
    int i;
    uint64_t rest;
    __device__ __forceinline__ Adapters(int id_, int j) : id(id_), i(-j), rest(__ballot(id_ >= 0)) {}
    // The next one and its tokens as a mask of lanes; false after the last.
    __device__ __forceinline__ bool next(int jn, int& ad, uint64_t& m) {
        while (rest) {
            ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
            m = __ballot(id == ad);
            rest &= ~m;
            const int k = i++;
            if (k >= 0 && k % jn == 0) return true;
        }
        return false;
    }
};
__device__ __forceinline__ int block_id(const LoraArgs& a, int t0, int tokens) {
    const int lane = threadIdx.x & 63, t = t0 + lane;
    const int id = lane < tokens && t < a.n ? a.ids[t] : -1;
    return id >= 0 && id < a.L ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs& a, int ad) {
    return a.ranks ? min(max(a.ranks[ad], 0), a.r) : a.r;
}

// part[split][t][:] = A[ids[t]][:, K of the split] x[t][K of the split]. A workgroup: 16 tokens,
// 16 RB ranks, one split. A is the MFMA's A operand (D row = rank), x its B (D column = token).
struct DownItem {
    int split, rank0, j, jn, t0, kb, ke;
    template <int RB>
    static __device__ __forceinline__ DownItem of(const LoraArgs& a) {
        DownItem d;
        int id = blockIdx.x;
        d.split = id % a.splits;
        id /= a.splits;
        const int rg = a.rp / 16 > RB ? (a.rp / 16 + RB - 1) / RB : 1;
        d.rank0 = id % rg * RB * 16;
        id /= rg;
        const BlockItem<1> b(a, id);
        d.t0 = b.t0, d.j = b.j, d.jn = b.jn;
        d.kb = d.split * a.kstep;
        d.ke = min(a.K, d.kb + a.kstep);
        return d;
    }
};

// Adds the waves' sums in order and stores those of the tokens in m, ranks from rk on as zeros.
template <int RB>
__device__ __forceinline__ void down_store(const LoraArgs& a, const DownItem& d, const f32x4 (&acc)[RB],
                                           f32x4 (*red)[RB][64], int rk, uint64_t m) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    __syncthreads();       // what red held before has been read
#pragma unroll
    for (int b = 0; b < RB; ++b) red[wv][b][lane] = acc[b];
    __syncthreads();
    for (int b = wv; b < RB; b += kLoraWaves) {
        const int row = d.rank0 + 16 * b + 4 * q;
        f32x4 v = red[0][b][lane];
#pragma unroll
        for (int w = 1; w < kLoraWaves; ++w) v += red[w][b][lane];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = row + c < rk ? v[c] : 0.0f;
        if (row < a.rp && (m >> r & 1))
            *reinterpret_cast<f32x4*>(a.part + ((long)d.split * a.n + d.t0 + r) * a.rp + row) = v;
    }
}

// Rows at any address: the waves take chunks of 64 of K in turn, straight to registers, the next chunk's
// loads before this one's products.
template <class W, class X, int RB>
__global__ __launch_bounds__(64 * kLoraWaves, 2) void lora_down_kernel(LoraArgs a) {
    constexpr int KS = 2, KC = 32 * KS;
    __shared__ f32x4 red[kLoraWaves][RB][64];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const DownItem d = DownItem::of<RB>(a);
    const typename X::row_t* xp =
        static_cast<const typename X::row_t*>(a.x) + (long)(d.t0 + r < a.n ? d.t0 + r : d.t0) * a.ldx;
    Adapters list(block_id(a, d.t0, 16), d.j);
    int ad;
    uint64_t m;
    while (list.next(d.jn, ad, m)) {
        const int rk = rank_of(a, ad);
        f32x4 acc[RB];
        const uint16_t* wp[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            // Rows past the adapter's ranks repeat its last one and are dropped.
            wp[b] = a.A + ((long)ad * a.r + max(min(d.rank0 + 16 * b + r, rk - 1), 0)) * a.K;
            acc[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        if (rk > d.rank0) {
            struct Chunk {
                u32x4 w[RB][KS];
                typename X::frag x[KS];
            };
            auto load = [&](Chunk& c, int k) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    c.x[s] = X::load(xp, k + 32 * s + 8 * q);
#pragma unroll
                    for (int b = 0; b < RB; ++b) c.w[b][s] = load8(wp[b], k + 32 * s + 8 * q);
                }
            };
            auto mul = [&](const Chunk& c) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const auto x = X::split(c.x[s]);
#pragma unroll
                    for (int b = 0; b < RB; ++b) acc[b] = X::mma(c.w[b][s], x, acc[b]);
                }
            };
            constexpr int STEP = KC * kLoraWaves;
            int k = d.kb + wv * KC;
            if (k + KC <= d.ke) {
                Chunk c0, c1;
                load(c0, k);
                for (;;) {
                    k += STEP;
                    const bool more = k + KC <= d.ke;
                    if (more) load(c1, k);
                    mul(c0);
                    if (!more) break;
                    k += STEP;
                    const bool more2 = k + KC <= d.ke;
                    if (more2) load(c0, k);
                    mul(c1);
                    if (!more2) break;
                }
            }
            if (k < d.ke) {
                Chunk c;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int kk = k + 32 * s + 8 * q;
                    c.x[s] = X::tail(xp, kk, d.ke);
#pragma unroll
                    for (int b = 0; b < RB; ++b) c.w[b][s] = load8_tail(wp[b], kk, d.ke);
                }
                mul(c);
            }
        }
        down_store<RB>(a, d, acc, red, rk, m);
    }
}

// The same for 16-byte aligned rows: steps of 128 of K come to LDS, x and A rows whole (256 or 512 B
// each), D steps in a ring; wave w has K 32 w .. 32 w + 31 of each step. Chunk c (16 B) of a
// row is at slot c ^ (row % 16): the 16 rows of a fragment fall on 16 different groups of banks. Two
// workgroups to a CU: with 32 tokens and one workgroup of twice the LDS, 4096 tokens of one adapter of rank
// 64, fp32 6144 -> 2048, took 56 us instead of 47.
template <class W, class X, int RB>
__global__ __launch_bounds__(64 * kLoraWaves, 2) void lora_down_ring_kernel(LoraArgs a) {
    constexpr int XB = sizeof(typename X::row_t), XROW = 128 * XB;
    constexpr int XN = 16 * XROW / 1024, AN = 16 * RB * 256 / 1024;          // instructions of a step
    constexpr int CX = XN / kLoraWaves, CA = AN / kLoraWaves, C = CX + CA, STEP = (XN + AN) * 1024;
    constexpr int D0 = 80 * 1024 / STEP, D = D0 < 8 ? D0 : 8;
    static_assert(CX * kLoraWaves == XN && CA * kLoraWaves == AN && D >= 3, "whole instructions");
    static_assert(kLoraWaves * RB * 1024 <= D * STEP, "the sums take the ring's place");
    __shared__ __align__(16) char lds[D * STEP];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const DownItem d = DownItem::of<RB>(a);
    const int steps = (d.ke - d.kb + 127) / 128;
    const uint32_t la = lds_addr(lds);

    // This lane's part of a copy: one chunk of row lane / (chunks of a row) of a piece of 1 KiB.
    constexpr int XL = XROW / 16, AL = 16;
    const char* px[CX];
    int kx[CX];                                    // the chunk's first K
#pragma unroll
    for (int i = 0; i < CX; ++i) {
        const int row = (kLoraWaves * i + wv) * (64 / XL) + lane / XL, tok = d.t0 + row;
        const int c = (lane % XL) ^ (row % 16);
        kx[i] = d.kb + c * 16 / XB;
        px[i] = static_cast<const char*>(a.x) + ((long)(tok < a.n ? tok : d.t0) * a.ldx + kx[i]) * XB;
    }
    Adapters list(block_id(a, d.t0, 16), d.j);
    int ad;
    uint64_t m;
    while (list.next(d.jn, ad, m)) {
        const int rk = rank_of(a, ad);
        f32x4 acc[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (rk > d.rank0) {
            const uint16_t* pa[CA];
            int ka[CA];
#pragma unroll
            for (int i = 0; i < CA; ++i) {
                // Rows past the adapter's ranks repeat its last one and are dropped.
                const int row = (kLoraWaves * i + wv) * 4 + lane / AL;
                ka[i] = d.kb + ((lane % AL) ^ (row % 16)) * 8;
                pa[i] = a.A + ((long)ad * a.r + min(d.rank0 + row, rk - 1)) * a.K + ka[i];
            }
            // Chunks past the split's K are zeros (K % 8 == 0: a chunk is inside or not).
            auto fetch = [&](int s, uint32_t slot) __attribute__((always_inline)) {
                const int k = s * 128;
#pragma unroll
                for (int i = 0; i < CX; ++i)
                    copy16(k + kx[i] < d.ke ? static_cast<const void*>(px[i] + k * XB) : &kZero16,
                           la + slot + (kLoraWaves * i + wv) * 1024);
#pragma unroll
                for (int i = 0; i < CA; ++i)
                    copy16(k + ka[i] < d.ke ? static_cast<const void*>(pa[i] + k) : &kZero16,
                           la + slot + XN * 1024 + (kLoraWaves * i + wv) * 1024);
            };
            __syncthreads();                       // the last adapter's sums are read
#pragma unroll
            for (int s = 0; s < D - 1; ++s)
                if (s < steps) fetch(s, s * STEP);
            uint32_t cur = 0, fill = (D - 1) * STEP;
            for (int s = 0; s < steps; ++s) {
                // Step s has arrived, and every wave has read step s - 1.
                if (s + D - 2 < steps)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n s_barrier" :: "n"((D - 2) * C) : "memory");
                else
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n s_barrier" ::: "memory");
                u32x4 w[RB];
                typename X::frag x;
                X::lds(lds + cur + r * XROW, 4 * wv + q, r, x);
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    w[b] = *reinterpret_cast<const u32x4*>(lds + cur + XN * 1024 + (16 * b + r) * 256 +
                                                           ((4 * wv + q) ^ r) * 16);
                if (s + D - 1 < steps) fetch(s + D - 1, fill);
                fill = cur;
                cur = cur + STEP == D * STEP ? 0 : cur + STEP;
                const auto xx = X::split(x);
#pragma unroll
                for (int b = 0; b < RB; ++b) acc[b] = X::mma(w[b], xx, acc[b]);
            }
        }
        down_store<RB>(a, d, acc, reinterpret_cast<f32x4 (*)[RB][64]>(lds), rk, m);
    }
}

// Element type of base and y: fp32 or a 16-bit type.
template <int DT>
struct Out {
    typedef uint16_t elem;
    static __device__ __forceinline__ float get(const elem* p) { return DT == kBf16 ? Bf16::up(*p) : F16::up(*p); }
    static __device__ __forceinline__ f32x4 get4(const elem* p) {
        const u32x2 w = *reinterpret_cast<const u32x2_any*>(p);
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = w[i / 2] >> (16 * (i & 1));
            v[i] = DT == kBf16 ? Bf16::up(u) : F16::up(u);
        }
        return v;
    }
    static __device__ __forceinline__ void put(elem* p, f32x4 v, int cnt) {
        if constexpr (DT == kBf16) store4<Bf16, false>(p, 0, v, cnt);
        else store4<F16, false>(p, 0, v, cnt);
    }
};
template <>
struct Out<kF32> {
    typedef float elem;
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ f32x4 get4(const float* p) { return *reinterpret_cast<const f32x4_any*>(p); }
    static __device__ __forceinline__ void put(float* p, f32x4 v, int cnt) { store4<Bf16, true>(p, 0, v, cnt); }
};

// y = base + scale * B (sum of part over the splits). A workgroup: 16 TB tokens, 256
// columns, 64 per wave; A x is summed, cut into three bf16 terms and kept in LDS, while the first
// adapter's rows of B and its tokens' base are on their way. B is the MFMA's A operand (D row =
// output), A x its B (D column = token): a lane has four neighbouring outputs of one token.
template <class W, int YD, int TB>
__global__ __launch_bounds__(64 * kLoraWaves, TB == 1 ? 4 : 2) void lora_up_kernel(LoraArgs a) {
    constexpr int NB = 4;
    typedef Out<YD> O;
    typedef typename O::elem elem;
    extern __shared__ __align__(16) uint16_t terms[];            // [3][16 TB][stride]
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4, stride = (a.r + 31) / 32 * 32 + 8;
    int id = blockIdx.x;
    const int n0 = (id % a.nx * kLoraWaves + wv) * 16 * NB;
    id /= a.nx;
    const BlockItem<TB> item(a, id);
    const int j = item.j, jn = item.jn, t0 = item.t0;
    const int left = min(a.n - t0, 16 * TB);
    const uint64_t here = left >= 64 ? ~0ull : (1ull << left) - 1;
    const int id0 = lane < left ? a.ids[t0 + lane] : -1;

    const int nl = n0 + 4 * q;                                   // the lane's first column
    const elem* pb = static_cast<const elem*>(a.base) + (long)(t0 + r) * a.ldb + nl;
    elem* py = static_cast<elem*>(a.y) + (long)(t0 + r) * a.ldy + nl;
    f32x4 base[TB][NB];
    u32x4 w[NB];
    const uint16_t* wp[NB];
    int rk = 0;
    auto load_w = [&](int k) __attribute__((always_inline)) {
        if (rk % 8 == 0) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                w[b] = (u32x4){0u, 0u, 0u, 0u};
                if (k + 8 * q < rk) w[b] = load8(wp[b], k + 8 * q);
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) w[b] = load8_tail(wp[b], k + 8 * q, rk);
        }
    };
    auto load_base = [&](uint64_t mask) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TB; ++t)
            if (mask >> (16 * t + r) & 1) {
                const elem* p = pb + 16L * t * a.ldb;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int cnt = a.N - nl - 16 * b;           // of its four columns, those inside N
                    if (cnt >= 4) {
                        base[t][b] = O::get4(p + 16 * b);
                    } else {
#pragma unroll
                        for (int c = 0; c < 3; ++c)
                            if (c < cnt) base[t][b][c] = O::get(p + 16 * b + c);
                    }
                }
            }
    };
    // The workgroups that all blocks have ask for the block's base and A x before they know its adapters.
    const int segs = stride / 8, tasks = 16 * TB * segs;
    const long step = (long)a.n * a.rp;
    auto load_part = [&](f32x4 (&u)[4][2], int i, int s) __attribute__((always_inline)) {
        const int t = min(i / segs, left - 1), k = min(i % segs * 8, a.rp - 8);
        const float* p = a.part + (long)(t0 + t) * a.rp + k;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const float* ps = p + min(s + d, a.splits - 1) * step;
            u[d][0] = *reinterpret_cast<const f32x4*>(ps);
            u[d][1] = *reinterpret_cast<const f32x4*>(ps + 4);
        }
    };
    f32x4 u[4][2];
    if (j == 0) {
        load_base(here);
        load_part(u, min((int)threadIdx.x, tasks - 1), 0);
    }
    const int ad0 = id0 >= 0 && id0 < a.L ? id0 : -1;
    const uint64_t has = __ballot(ad0 >= 0);
    Adapters list(ad0, j);
    int ad;
    uint64_t m;
    bool some = list.next(jn, ad, m);
    // Tokens without an adapter are copied; in place they are there already.
    const uint64_t none = j == 0 && a.y != a.base ? ~has & here : 0;
    if (!some && !none) return;
    auto begin = [&]() __attribute__((always_inline)) {
        rk = rank_of(a, ad);
#pragma unroll
        for (int b = 0; b < NB; ++b) wp[b] = a.B + ((long)ad * a.N + min(n0 + 16 * b + r, a.N - 1)) * a.r;
        load_w(0);
        if (j != 0) load_base(m);
    };
    if (some) begin();

    for (int i = threadIdx.x; i < tasks; i += 64 * kLoraWaves) {
        const int t = i / segs, k = i % segs * 8;
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = 0.0f;
        for (int s = 0; s < a.splits; s += 4) {
            if (j != 0 || s > 0 || i >= 64 * kLoraWaves) load_part(u, i, s);
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = s + d < a.splits ? v[c] + u[d][c / 4][c % 4] : v[c];
        }
        // Rows of tokens without an adapter, and what lies past the ranks, hold nothing.
        const bool live = k < a.rp && (has >> t & 1);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = live ? v[c] : 0.0f;
        const Terms3 o = split3(v);
#pragma unroll
        for (int c = 0; c < 3; ++c) *reinterpret_cast<u32x4*>(terms + (c * 16 * TB + t) * stride + k) = o.t[c];
    }
    __syncthreads();

    while (some) {
        const float sc = a.scale ? a.scale[ad] : 1.0f;
        f32x4 acc[NB][TB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[b][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < rk; k += 32) {
            if (k) load_w(k);
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                Terms3 x;
#pragma unroll
                for (int c = 0; c < 3; ++c)
                    x.t[c] = *reinterpret_cast<const u32x4*>(terms + ((c * TB + t) * 16 + r) * stride + k + 8 * q);
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b][t] = mma3<W>(w[b], x, acc[b][t]);
            }
        }
#pragma unroll
        for (int t = 0; t < TB; ++t)
            if (m >> (16 * t + r) & 1) {
                elem* p = py + 16L * t * a.ldy;
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    if (nl + 16 * b < a.N) {
                        f32x4 v;
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[c] = __builtin_fmaf(sc, acc[b][t][c], base[t][b][c]);
                        O::put(p + 16 * b, v, a.N - nl - 16 * b);
                    }
            }
        some = list.next(jn, ad, m);
        if (some) begin();
    }
    if (none) {
#pragma unroll
        for (int t = 0; t < TB; ++t)
            if (none >> (16 * t + r) & 1) {
                elem* p = py + 16L * t * a.ldy;
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    if (nl + 16 * b < a.N) O::put(p + 16 * b, base[t][b], a.N - nl - 16 * b);
            }
    }
}

// How the first launch splits K: into 512 workgroups (1024: 4096 tokens of 8 adapters of rank 64, fp32
// 6144 -> 2048, 62 us against 64, but one adapter 51 against 47 and 64 decoding tokens of 32 adapters 26.7
// against 23.5; 256: 75 for the first), 512 of K at least.
constexpr int kDownGroups = 512;
struct LoraPlan {
    int jm, je, splits, kstep, rp;
};
static LoraPlan plan_of(int n, int L, int K, int r) {
    LoraPlan p;
    const int most = n < L ? n : L;
    // A workgroup that finds no adapter costs its start: up to 256 tokens may all be decoding, beyond
    // most are prompts' (2048 tokens of 4 prompts, rank 16, bf16 6144 -> 6144: 35 us with two workgroups for
    // every block, 33 with one; 700 tokens of 3 prompts and 32 decoding: 22 with 16 for every block, 18
    // with four).
    const int jm = n <= 256 ? 16 : n <= 1024 ? 4 : 1;
    p.je = most < 16 ? most : 16;
    p.jm = p.je < jm ? p.je : jm;
    p.rp = (r + 15) / 16 * 16;
    const long wgs = (long)BlockItem<1>::blocks(n) * (n <= 256 ? p.jm : 1) *
                     ((r + 16 * kRankBlocks - 1) / (16 * kRankBlocks));
    long s = (kDownGroups + wgs - 1) / wgs;
    const int top = (K + 511) / 512;
    s = s < 1 ? 1 : s > top ? top : s;
    p.kstep = (int)(((K + s - 1) / s + 127) / 128 * 128);
    p.splits = (K + p.kstep - 1) / p.kstep;
    return p;
}
// What any plan of these sizes or smaller ones takes: splits < kDownGroups / wgs + 1 and wgs >= n / 16, so splits * n
// < 16 kDownGroups + n; and no more than K's own limit. A plan's own need is not monotone (8176 tokens
// have two splits, 8192 one), and a workspace for the most tokens has to serve fewer.
size_t lora_part_bytes(int n, int K, int r) {
    const size_t all = (size_t)n * ((K + 511) / 512), most = (size_t)16 * kDownGroups + n;
    return (all < most ? all : most) * ((r + 15) / 16 * 16) * 4;
}

template <class W, class X>
static void run_down(const LoraArgs& a, const LoraPlan& p, bool aligned, unsigned grid, hipStream_t s) {
    const dim3 g(grid), b(64 * kLoraWaves);
    const int rb = p.rp / 16;
    auto go = [&](auto r) {
        constexpr int RB = decltype(r)::value;
        if (aligned) hipLaunchKernelGGL((lora_down_ring_kernel<W, X, RB>), g, b, 0, s, a);
        else hipLaunchKernelGGL((lora_down_kernel<W, X, RB>), g, b, 0, s, a);
    };
    if (rb == 1) go(std::integral_constant<int, 1>{});
    else if (rb == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
}

template <class W, int YD>
static int run_up(const LoraArgs& a0, hipStream_t s) {
    LoraArgs a = a0;
    const int tb = a.n > 1024 ? 2 : 1;
    a.nx = (a.N + 255) / 256;
    const long grid = (tb == 1 ? BlockItem<1>::count(a) : BlockItem<2>::count(a)) * a.nx;
    if (grid * 64 * kLoraWaves >= (1L << 32)) return -2;   // threads of a launch
    const size_t lds = (size_t)3 * 16 * tb * ((a.r + 31) / 32 * 32 + 8) * 2;
    const dim3 g((unsigned)grid), b(64 * kLoraWaves);
    if (tb == 1) hipLaunchKernelGGL((lora_up_kernel<W, YD, 1>), g, b, lds, s, a);
    else hipLaunchKernelGGL((lora_up_kernel<W, YD, 2>), g, b, lds, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int launch_lora(const LoraArgs& a0, int xdt, int wdt, int ydt, hipStream_t s) {
    LoraArgs a = a0;
    const LoraPlan p = plan_of(a.n, a.L, a.K, a.r);
    a.splits = p.splits, a.kstep = p.kstep, a.rp = p.rp, a.jm = p.jm, a.je = p.je;
    auto al = [](const void* q, size_t v) { return reinterpret_cast<uintptr_t>(q) % v == 0; };
    const bool aligned = a.K % 8 == 0 && al(a.x, 16) && al(a.A, 16) && a.ldx % (xdt == kF32 ? 4 : 8) == 0;
    const long grid = BlockItem<1>::count(a) * ((p.rp / 16 + kRankBlocks - 1) / kRankBlocks) * p.splits;
    if (grid * 64 * kLoraWaves >= (1L << 32)) return -2;   // threads of a launch
    auto down = [&](auto w) {
        using W = decltype(w);
        const unsigned g = (unsigned)grid;
        if (xdt == kF32) run_down<W, XFloat<W>>(a, p, aligned, g, s);
        else run_down<W, XHalf<W>>(a, p, aligned, g, s);
    };
    if (wdt == kBf16) down(Bf16{});
    else down(F16{});
    if (hipGetLastError() != hipSuccess) return -4;
    if (wdt == kBf16) return ydt == kF32 ? run_up<Bf16, kF32>(a, s) : run_up<Bf16, kBf16>(a, s);
    return ydt == kF32 ? run_up<F16, kF32>(a, s) : run_up<F16, kF16>(a, s);
}

}  // namespace glmmoe
