// Attention over blocks of 64 keys that a cheap score selects for each query, forward and backward.
//
//   bounds    per block and kv head: upper / lower bound of every channel over the visible keys, as integers U, L (fp16) times one scale s_j
//   score     sum_g sum_d (q_d > 0 ? q_d U_d : q_d L_d) s_j,  q as integers up to 127: an upper bound of q . k in the block.  Every partial
//             sum is an integer below 2^24 (G D 127^2 with G D <= 1024): the fp16 matrix instruction adds it without rounding, so the
//             choice is the same whoever computes it
//   select    the n largest scores, ties to the lowest block, ascending
//   attend    softmax over the visible keys of a query's blocks; a query with none gets zeros
//
// Each query has blocks of its own, so a tile of neighbouring queries shares none: read query by query, K and V would cross the L2 once per
// (query, block).  With many queries the work is turned round: the mentions of a block are listed (a counting sort that keeps their order),
// one workgroup holds the block's K and V in LDS and takes the queries that named it through matrix instructions, 32 per wave; every mention
// writes its (o, max, sum) to a place of its own and a second pass joins the n places of a query.  No atomics: dK and dV of a block are summed
// by the workgroups that hold it, in the order of its list.  With few queries one wave takes one mention and reads its block directly.
#include <algorithm>
#include <type_traits>

#include "token_common.hpp"

namespace {

constexpr int kKeys = 64;                    // keys of a block
constexpr int kMaxPick = 64;                 // blocks a query may have
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTinyBs = 1e-30f;
constexpr float kHugeBs = 1e32f;             // keys and queries beyond it, infinities too, count as it: every score is a number (2^24 kHugeBs / 127 < FLT_MAX)

template <typename T> struct is_f32 : std::false_type {};
template <> struct is_f32<float> : std::true_type {};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct BsArgs {
    const void *q, *k, *v;
    const uint8_t* mask;                     // (B, Nk) visible keys, or null
    const int32_t* blocks;                   // (B, T, KV, n)
    long long qb, qt, qh, kb, kt, kh, vb, vt, vh;      // element strides
    int B, T, Nk, H, KV, G, NB, n;
    float scale;
    // lists
    const int32_t* list;                     // (B KV, T n) mentions t * 64 + slot of block 0, 1, ..
    const int32_t* start;                    // (B KV, NB + 1)
    const int32_t* items;                    // (B KV, max_items) 2 x int32: block, first row
    const int32_t* n_items;                  // (B KV)
    int max_items, item_rows;
    // forward
    void* part;                              // forward: (B, T, H, n) records; backward: (B, T, H, n, D) fp32, dQ
    void* out;                               // (B, T, H, D)
    float* lse;                              // (B, T, H) base 2, +inf: no key; may be null
    void* rest;                              // (B, T, H, D) out's rounding errors, or null
    // backward
    const void* dout;
    const f32x2* ld;                         // (B, T, H) log-sum-exp (base 2), sum dO O
    float* slab;                             // (B KV, max_items, 2, 64, D)
    void *dq, *dk, *dv;
};

// ------------------------------------------------------------------------------------------------------------ bounds
// One wave per (block, kv head): D / 4 lanes a key, 256 / D keys a step.  Bound by HBM: K is read once (140800 keys x 8 heads of 32, bf16: 15 us, 4.7 TB/s; 26 us where each
// load waits for its key's mask).
template <typename T, int D>
__global__ __launch_bounds__(256) void bs_bounds_kernel(const T* __restrict__ k, const uint8_t* __restrict__ mask, long long kb, long long kt, long long kh,
                                                        int nk, int kv, int nb, int first, int count, _Float16* __restrict__ ints, float* __restrict__ scale,
                                                        long long total) {
    constexpr int LPK = D / 4, KPS = 64 / LPK;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= total) return;
    const int lane = threadIdx.x & 63, sub = lane % LPK;
    const int h = (int)(w % kv), j = first + (int)(w / kv % count), b = (int)(w / kv / count);
    const int key = j * kKeys + lane;
    const unsigned long long seen = __ballot(key < nk && (!mask || mask[(size_t)b * nk + key]));
    const int one = seen ? __ffsll(seen) - 1 : 0;        // stands in for keys that are not visible: all loads are in flight together
    const bool some = seen != 0;
    f32x4 hi{-INFINITY, -INFINITY, -INFINITY, -INFINITY}, lo{INFINITY, INFINITY, INFINITY, INFINITY};
    if (some) {
        const T* p = k + b * kb + (long long)j * kKeys * kt + h * kh + sub * 4;
#pragma unroll
        for (int s = 0; s < kKeys / KPS; ++s) {
            const int t = s * KPS + lane / LPK;
            const f32x4 x = tok_load4(p + (seen >> t & 1 ? t : one) * kt);
#pragma unroll
            for (int i = 0; i < 4; ++i) { hi[i] = fmaxf(hi[i], x[i]); lo[i] = fminf(lo[i], x[i]); }
        }
    }
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], o)); lo[i] = fminf(lo[i], __shfl_xor(lo[i], o)); }
    }
    if (!some) hi = lo = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
#pragma unroll
    for (int o = 1; o < LPK; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    m = fminf(m, kHugeBs);
    const float r = 127.0f / fmaxf(m, kTinyBs);
    if (lane < LPK) {
        const size_t at = ((size_t)b * kv + h) * nb + j;
        typename tok_vec<_Float16>::v4 u, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = (_Float16)fminf(fmaxf(rintf(hi[i] * r), -127.f), 127.f);
            l[i] = (_Float16)fminf(fmaxf(rintf(lo[i] * r), -127.f), 127.f);
        }
        *reinterpret_cast<typename tok_vec<_Float16>::v4*>(ints + at * 2 * D + sub * 4) = u;
        *reinterpret_cast<typename tok_vec<_Float16>::v4*>(ints + at * 2 * D + D + sub * 4) = l;
        if (lane == 0) scale[at] = some ? m / 127.0f : -1.0f;
    }
}

// ------------------------------------------------------------------------------------------------------------ selection
constexpr int kChunk = 512;                  // scores of 16 queries in LDS
constexpr int kScPitch = kChunk + 4;         // 4 consecutive scores per store, 16 queries: all banks

__device__ __forceinline__ unsigned order_key(float s) {       // unsigned order of floats; 0 = not a candidate
    const int b = __builtin_bit_cast(int, s + 0.0f);
    return (unsigned)(b < 0 ? b ^ 0x7fffffff : b) ^ 0x80000000u;
}

__device__ __forceinline__ float key_score(unsigned k) {       // the score of a key; the key below zero's (-0, which no score has) is that of the number below zero
    if (k == 0x7fffffffu) k = 0x7ffffffeu;
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// n largest of {key (lane), c[0], c[1], ..} (candidates in this order, lane by lane), 0 = none, ties to the earliest.  Returns how many; the
// chosen ones land in key / idx of lanes 0, 1, .. in order.  Any number of ties: the n-th largest value is found bit by bit.
template <int E, typename Idx>
__device__ __forceinline__ int keep_largest(unsigned& key, int& idx, const unsigned (&c)[E], Idx&& index, int n, unsigned* lk, int* li, int lane) {
    unsigned t = 0;
    bool exact = false;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = t | 1u << bit;
        int cnt = __popcll(__ballot(key >= trial));
#pragma unroll
        for (int e = 0; e < E; ++e) cnt += __popcll(__ballot(c[e] >= trial));
        if (cnt >= n) t = trial;
        if (cnt == n) { exact = true; break; }
    }
    // t: the n-th largest (0: fewer than n candidates), or a bound that exactly n reach
    int above = 0;
    if (!exact) {
        above = __popcll(__ballot(key > t));
#pragma unroll
        for (int e = 0; e < E; ++e) above += __popcll(__ballot(c[e] > t));
    }
    int ties = exact || t == 0 ? 0 : n - above, out = 0;
    const unsigned long long below = (1ull << lane) - 1;
    auto put = [&](unsigned x, int i) {
        const unsigned long long eq = __ballot(!exact && t != 0 && x == t);
        const bool in = exact ? x >= t : x > t || (x == t && t != 0 && __popcll(eq & below) < ties);
        const unsigned long long m = __ballot(in);
        if (in) { lk[out + __popcll(m & below)] = x; li[out + __popcll(m & below)] = i; }
        ties -= min(ties, __popcll(eq));
        out += __popcll(m);
    };
    put(key, idx);
#pragma unroll
    for (int e = 0; e < E; ++e) put(c[e], index(e));
    __builtin_amdgcn_wave_barrier();
    key = lane < out ? lk[lane] : 0u;
    idx = lane < out ? li[lane] : -1;
    __builtin_amdgcn_wave_barrier();
    return out;
}

// The same for a few newcomers: candidates above `least` join the kept ones in LDS (at most 64 together), every one counts how many are better, and the
// n best stay, in order.  Returns false where they are too many (the caller goes bit by bit).
template <int E, typename Idx>
__device__ __forceinline__ bool merge_few(unsigned& key, int& idx, int& have, unsigned& least, const unsigned (&c)[E], Idx&& index, int n, unsigned* lk, int* li, int lane) {
    unsigned long long m[E];
    int total = have;
#pragma unroll
    for (int e = 0; e < E; ++e) { m[e] = __ballot(c[e] > least); total += __popcll(m[e]); }
    if (total == have) return true;
    if (total > 64) return false;
    int at = have;
    if (lane < have) { lk[lane] = key; li[lane] = idx; }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (m[e]) {
            const int p = at + __builtin_amdgcn_mbcnt_hi((unsigned)(m[e] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m[e], 0));
            if (c[e] > least) { lk[p] = c[e]; li[p] = index(e); }
            at += __popcll(m[e]);
        }
    }
    __builtin_amdgcn_wave_barrier();
    unsigned k = lane < total ? lk[lane] : 0u;
    int x = lane < total ? li[lane] : -1;
    if (total > n) {
        int rank = 0;           // how many are better: larger, or equal and earlier
        for (int i = 0; i < total; ++i) {
            const unsigned o = __builtin_amdgcn_readlane(k, i);
            rank += o > k || (o == k && i < lane) ? 1 : 0;
        }
        const unsigned long long in = __ballot(lane < total && rank < n), last = __ballot(lane < total && rank == n - 1);
        least = __builtin_amdgcn_readlane(k, __ffsll(last) - 1);
        __builtin_amdgcn_wave_barrier();
        if (lane < total && rank < n) {
            const int p = __builtin_amdgcn_mbcnt_hi((unsigned)(in >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)in, 0));
            lk[p] = k;
            li[p] = x;
        }
        __builtin_amdgcn_wave_barrier();
        total = n;
        k = lane < n ? lk[lane] : 0u;
        x = lane < n ? li[lane] : -1;
    } else if (total == n) {
        least = lane < n ? k : 0xffffffffu;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) least = min(least, (unsigned)__shfl_xor((int)least, o));
    }
    __builtin_amdgcn_wave_barrier();
    key = k;
    idx = x;
    have = total;
    return true;
}

// the kept n and E x 64 newcomers; least: the smallest kept one once n are kept
template <int E, typename Idx>
__device__ __forceinline__ void take(unsigned& key, int& idx, int& have, unsigned& least, const unsigned (&c)[E], Idx&& index, int n, unsigned* lk, int* li, int lane) {
    if (have < n) {
        // nothing to compare with yet: the n-th largest of the group maxima is a bound that at least n candidates reach, and few more
        unsigned g = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) g = max(g, c[e]);
        const int step = n <= 16 ? 4 : 1;
        if (n <= 16) {
            g = max(g, (unsigned)__shfl_xor((int)g, 1));
            g = max(g, (unsigned)__shfl_xor((int)g, 2));
        }
        int rank = 0;
        for (int i = 0; i < 64; i += step) {
            const unsigned o = __builtin_amdgcn_readlane(g, i);
            rank += o > g || (o == g && i < lane) ? 1 : 0;
        }
        const unsigned long long at = __ballot(rank == n - 1 && lane % step == 0);
        const unsigned t = at ? __builtin_amdgcn_readlane(g, __ffsll(at) - 1) : 0u;
        least = have == 0 && t > 0 ? t - 1 : 0u;
    }
    if (!merge_few(key, idx, have, least, c, index, n, lk, li, lane)) {
        have = keep_largest(key, idx, c, index, n, lk, li, lane);
        least = 0u;
        if (have == n) {
            least = lane < n ? key : 0xffffffffu;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) least = min(least, (unsigned)__shfl_xor((int)least, o));
        }
    } else if (have < n) {
        least = 0u;
    }
}

// 16 queries x 1 kv head x a range of blocks a workgroup: integers of the queries, scores of 512 blocks at a time on the fp16 matrix cores, the n best kept in
// a wave's registers (four queries a wave).  PARTS: the range is one of several, its n best go to `part` as (key, block) pairs.
template <typename T, int D, bool PARTS>
__global__ __launch_bounds__(256) void bs_select_kernel(const T* __restrict__ q, long long qb, long long qt, long long qh, const _Float16* __restrict__ ints,
                                                        const float* __restrict__ scale, int T_, int G, int KV, int NB, int n, int parts, int per, int32_t* __restrict__ out,
                                                        uint2* __restrict__ part) {
    __shared__ __align__(16) unsigned sc[16 * kScPitch];
    __shared__ __align__(16) _Float16 qi[16][2 * D + 8];
    __shared__ unsigned lk[4][64];
    __shared__ int li[4][64];
    constexpr int CH = D / 16, KS = 2 * D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int t0 = (PARTS ? blockIdx.x / parts : blockIdx.x) * 16, h = blockIdx.y, b = blockIdx.z;
    const int first = PARTS ? (blockIdx.x % parts) * per : 0, last = PARTS ? min(NB, first + per) : NB;
    {
        const int row = tid >> 4, l = tid & 15, t = min(t0 + row, T_ - 1);
        const T* p = q + b * qb + t * qt + (long long)h * G * qh + l * CH;
        float m = 0.f;
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int c = 0; c < CH; ++c) m = fmaxf(m, fabsf((float)p[g * qh + c]));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float r = 127.0f / fminf(fmaxf(m, kTinyBs), kHugeBs);
        float up[CH], lo[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) up[c] = lo[c] = 0.f;
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float x = fminf(fmaxf(rintf((float)p[g * qh + c] * r), -127.f), 127.f);
                up[c] += fmaxf(x, 0.f);
                lo[c] += fminf(x, 0.f);
            }
#pragma unroll
        for (int c = 0; c < CH; ++c) {       // at most 127 G <= 2048: exact in fp16
            qi[row][l * CH + c] = (_Float16)up[c];
            qi[row][D + l * CH + c] = (_Float16)lo[c];
        }
    }
    __syncthreads();
    f16x8 bf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) bf[s] = *reinterpret_cast<const f16x8*>(&qi[lane & 15][s * 32 + (lane >> 4) * 8]);
    const _Float16* kp = ints + ((size_t)b * KV + h) * NB * 2 * D;
    const float* sp = scale + ((size_t)b * KV + h) * NB;
    unsigned key[4] = {0u, 0u, 0u, 0u}, least[4] = {0u, 0u, 0u, 0u};
    int idx[4] = {-1, -1, -1, -1}, have[4] = {0, 0, 0, 0};
    for (int j0 = first; j0 < last; j0 += kChunk) {
        const int tiles = (min(kChunk, last - j0) + 15) / 16;
        for (int tl = wave; tl < kChunk / 16; tl += 4) {
            const int jr = j0 + tl * 16;
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
            if (tl < tiles) {
                const int ja = min(jr + (lane & 15), NB - 1);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const f16x8 a = *reinterpret_cast<const f16x8*>(kp + (size_t)ja * 2 * D + s * 32 + (lane >> 4) * 8);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bf[s], acc, 0, 0, 0);
                }
            }
            unsigned k4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = jr + (lane >> 4) * 4 + i;
                const float s = j < last ? sp[j] : -1.0f;
                k4[i] = s < 0.f ? 0u : order_key(acc[i] * s);
            }
            *reinterpret_cast<uint4*>(&sc[(lane & 15) * kScPitch + tl * 16 + (lane >> 4) * 4]) = make_uint4(k4[0], k4[1], k4[2], k4[3]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned c[kChunk / 64];
#pragma unroll
            for (int e = 0; e < kChunk / 64; ++e) c[e] = sc[(wave * 4 + u) * kScPitch + e * 64 + lane];
            take(key[u], idx[u], have[u], least[u], c, [&](int e) { return j0 + e * 64 + lane; }, n, lk[wave], li[wave], lane);
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int t = t0 + wave * 4 + u;
        if (t >= T_ || lane >= n) continue;
        const size_t at = ((size_t)b * T_ + t) * KV + h;
        if constexpr (PARTS) part[(at * parts + blockIdx.x % parts) * n + lane] = lane < have[u] ? make_uint2(key[u], (unsigned)idx[u]) : make_uint2(0u, 0xffffffffu);
        else out[at * n + lane] = lane < have[u] ? idx[u] : -1;
    }
}

// The same for n <= 16, the common case: 32 queries a workgroup.  The scores themselves are not kept: the matrix cores' tile leaves the largest of every four
// blocks in LDS (1536 blocks at a time, 50 KB), sixteen lanes a query look for the fours above the n-th best so far -- at first above the n-th largest of
// the lanes' own maxima, which at least n scores reach -- and only their scores are computed again, exactly, one a lane.  What is above goes to a list of
// pending entries; sixteen at a time count how many of the kept and of each other are better, which is their place.  Loops, not unrolled
// code: an unrolled form of this filled the instruction cache (10 000 instructions) and ran at 1490 us.  281600 queries x 2200 blocks of 32 channels, bf16, n = 8:
// 520 us, 1.2e12 scores a second.  Counters: vector instructions issue in 60 % of the cycles, the matrix cores are busy in 7 %, and a wave waits two thirds of its time
// (LDS, L2, barriers; four waves a SIMD, 8 % of the cycles lost to bank conflicts of the picking).  L2 serves 31 million requests of at most 128 bytes (the bounds,
// once for every 32 queries, and the picking's), 120 us at the 34 TB/s that this path reaches: vector issue and the waits between short phases bound it, not L2.
// Without the picking it takes two thirds; the matrix products are 33 us.  64 queries a workgroup halve those bytes but leave one workgroup a CU, whose scores and
// picks no longer overlap (568 us against 479 under the same clock); the next tiles fetched ahead gained nothing.  n = 1 / 8 / 16: 408 / 478 / 584 us where the kernel
// above takes 1075 / 1650 / 1812; 35200 queries of 2 x 64 channels x 550 blocks: 78 / 96 / 125 and 178 / 266 / 269; one query x 2200 blocks: 11 / 13 / 21 and 28 / 28 / 28.
template <int R> __device__ __forceinline__ unsigned row_ror(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + R, 0xf, 0xf, false);
}
template <int R, int N, typename F> __device__ __forceinline__ void each_ror(F&& f) {
    if constexpr (R < N) {
        f(std::integral_constant<int, R>{});
        each_ror<R + 1, N>(f);
    }
}
template <int CTRL> __device__ __forceinline__ float dpp_f(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ int row_sum(int x) {
    x += (int)row_ror<8>((unsigned)x);
    x += (int)row_ror<4>((unsigned)x);
    x += (int)row_ror<2>((unsigned)x);
    return x + (int)row_ror<1>((unsigned)x);
}
__device__ __forceinline__ int rows_max(int x) {       // the largest of four rows' values, in a scalar
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)), max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}

constexpr int kFours = 384;                  // fours of blocks in LDS: six steps of 64, four bits of a word each
constexpr int kGroupList = 64;               // fours of a query that are looked at in one go

typedef unsigned long long u64;
typedef u64 u64x2 __attribute__((ext_vector_type(2)));

template <typename T, int D, bool PARTS>
__global__ __launch_bounds__(512, (D <= 64 ? 4 : 2)) void bs_select16_kernel(const T* __restrict__ q, long long qb, long long qt, long long qh, const _Float16* __restrict__ ints,
                                                             const float* __restrict__ scale, int T_, int G, int KV, int NB, int n, int parts, int per,
                                                             int32_t* __restrict__ out, uint2* __restrict__ part) {
    constexpr int NQ = 32, CH = D / 16, KS = 2 * D / 32, GT = KS <= 2 ? 4 : KS <= 4 ? 2 : 1, GP = kFours + 4, QP = 2 * D + 8;
    constexpr int LB = D <= 64 ? D / 4 : 16, CPL = D <= 64 ? 1 : 2;      // lanes that add up one score, 16-byte pieces of each
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    __shared__ __align__(16) float gm[NQ * GP];                                // the largest score of every four, -inf: no block
    __shared__ __align__(16) _Float16 qi[NQ * QP];
    // entries: key of the score in the upper half, ~block in the lower one: larger is better, ties to the lower block; 0: none
    __shared__ __align__(16) u64 kept[NQ][16], pend[NQ][32];
    __shared__ __align__(16) unsigned short fours[NQ][kGroupList];               // before them, in the same bytes: 32 maxima of a query's scores
    static_assert(sizeof(fours[0]) == 32 * sizeof(float), "one row of maxima");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane & 15, row = lane >> 4;
    const int t0 = (PARTS ? blockIdx.x / parts : blockIdx.x) * NQ, h = blockIdx.y, b = blockIdx.z;
    const int first = PARTS ? (blockIdx.x % parts) * per : 0, last = PARTS ? min(NB, first + per) : NB;
    for (int i = tid; i < NQ * 32; i += 512) { (&pend[0][0])[i] = 0ull; if (i < NQ * 16) (&kept[0][0])[i] = 0ull; }
    {
        const int r8 = tid >> 4, l8 = tid & 15, t = min(t0 + r8, T_ - 1);
        const T* p = q + b * qb + t * qt + (long long)h * G * qh + l8 * CH;
        float m = 0.f;
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int c = 0; c < CH; ++c) m = fmaxf(m, fabsf((float)p[g * qh + c]));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float r = 127.0f / fminf(fmaxf(m, kTinyBs), kHugeBs);
        float up[CH], lo[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) up[c] = lo[c] = 0.f;
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float x = fminf(fmaxf(rintf((float)p[g * qh + c] * r), -127.f), 127.f);
                up[c] += fmaxf(x, 0.f);
                lo[c] += fminf(x, 0.f);
            }
#pragma unroll
        for (int c = 0; c < CH; ++c) {       // at most 127 G <= 2048: exact in fp16
            qi[r8 * QP + l8 * CH + c] = (_Float16)up[c];
            qi[r8 * QP + D + l8 * CH + c] = (_Float16)lo[c];
        }
    }
    __syncthreads();
    const _Float16* kp = ints + ((size_t)b * KV + h) * NB * 2 * D;
    const float* sp = scale + ((size_t)b * KV + h) * NB;
    const int qr = wave * 4 + row;           // this row's query
    u64* pe = pend[qr];
    unsigned short* fo = fours[qr];
    f16x8 y[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) y[c] = *reinterpret_cast<const f16x8*>(&qi[qr * QP + (l % LB + c * LB) * 8]);
    for (int j0 = first; j0 < last; j0 += kFours * 4) {
        const int tiles = (min(kFours * 4, last - j0) + 15) / 16, steps = (tiles + 15) / 16;       // 16 tiles: 64 fours, four a lane
        {
            f16x8 bf[2][KS];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int s = 0; s < KS; ++s) bf[u][s] = *reinterpret_cast<const f16x8*>(&qi[(u * 16 + l) * QP + s * 32 + row * 8]);
            float mx[2] = {-INFINITY, -INFINITY};                                 // over this wave's blocks, one row's share of each tile
            // a wave takes GT neighbouring tiles at a time; tiles too few for all waves go round them one by one, so that every row has maxima for the first bound
            // (4400 queries x 138 blocks, n = 8 / 16: 26 / 36 us, 33 / 55 with neighbouring tiles; 35200 x 550, n = 8: 218 and 211 the other way)
            const bool spread = steps * 16 < 8 * GT;
            const int gs = spread ? 8 : 1;
            for (int g0 = spread ? wave : wave * GT; g0 < steps * 16; g0 += 8 * GT) {
                f16x8 a[GT][KS];
                f32x4 w[GT], none[GT];                                            // score = dot * w + none: -inf where there is no block
                const int jr = j0 + g0 * 16;
                if (!spread && jr + GT * 16 <= last) {
                    const _Float16* p = kp + (unsigned)((jr + l) * 2 * D + row * 8);
#pragma unroll
                    for (int g = 0; g < GT; ++g) {
#pragma unroll
                        for (int s = 0; s < KS; ++s) a[g][s] = *reinterpret_cast<const f16x8*>(p + g * 16 * 2 * D + s * 32);
                        __builtin_memcpy(&w[g], sp + jr + g * 16 + row * 4, 16);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < GT; ++g) {
                        const int jg = jr + g * gs * 16, ja = min(jg + l, NB - 1);
#pragma unroll
                        for (int s = 0; s < KS; ++s) a[g][s] = *reinterpret_cast<const f16x8*>(kp + (unsigned)(ja * 2 * D + s * 32 + row * 8));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = jg + row * 4 + i;
                            const float x = sp[min(j, NB - 1)];
                            w[g][i] = j < last ? x : -1.0f;
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < GT; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        none[g][i] = w[g][i] < 0.f ? -INFINITY : 0.f;
                        w[g][i] = fmaxf(w[g][i], 0.f);
                    }
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const int tile = g0 + g * gs;
                    if (tile >= steps * 16) break;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[g][s], bf[u][s], acc, 0, 0, 0);
                        float m = fmaf(acc[0], w[g][0], none[g][0]);
#pragma unroll
                        for (int i = 1; i < 4; ++i) m = fmaxf(m, fmaf(acc[i], w[g][i], none[g][i]));
                        gm[(u * 16 + l) * GP + tile * 4 + row] = m;
                        mx[u] = fmaxf(mx[u], m);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) reinterpret_cast<float*>(fours[u * 16 + l])[wave * 4 + row] = mx[u];
        }
        __syncthreads();
        if (t0 + wave * 4 < T_) {
            const float* gp = gm + qr * GP + l * 4;
            u64 k = kept[qr][l];
            // what an entry has to beat: the n-th best (a block of this range may tie with it and come first), or every entry of a key
            u64 bar = kept[qr][n - 1];
            const bool none = kept[qr][0] == 0ull;
            if (__ballot(none)) {
                const f32x2 m = *reinterpret_cast<const f32x2*>(&fo[l * 4]);
                const unsigned ma = m.x == -INFINITY ? 0u : order_key(m.x), mb = m.y == -INFINITY ? 0u : order_key(m.y);
                int ra = mb > ma ? 1 : 0, rb = ma > mb ? 1 : 0;
                each_ror<1, 16>([&](auto r) {
                    const unsigned oa = row_ror<decltype(r)::value>(ma), ob = row_ror<decltype(r)::value>(mb);
                    ra += (oa > ma ? 1 : 0) + (ob > ma ? 1 : 0);
                    rb += (oa > mb ? 1 : 0) + (ob > mb ? 1 : 0);
                });
                unsigned t = min(ra < n ? ma : 0xffffffffu, rb < n ? mb : 0xffffffffu);
                t = min(t, row_ror<8>(t));
                t = min(t, row_ror<4>(t));
                t = min(t, row_ror<2>(t));
                t = min(t, row_ror<1>(t));
                if (none && t > 0) bar = (u64)(t - 1) << 32 | 0xffffffffu;
                __builtin_amdgcn_wave_barrier();
            }
            int pc = 0;
            // sixteen pending entries of every row enter; a loop over what is kept and what is new, two at a time
            auto flush = [&]() {
                const u64 x = pe[l];
                const int have = __popc((unsigned)(__ballot(k != 0ull) >> (row * 16)) & 0xffffu);
                int rk = l, rx = 0;
                for (int i = 0; i < n; i += 4) {
                    const u64x2 y = *reinterpret_cast<const u64x2*>(&kept[qr][i]), z = *reinterpret_cast<const u64x2*>(&kept[qr][i + 2]);
                    rx += (y[0] > x ? 1 : 0) + (y[1] > x ? 1 : 0) + (z[0] > x ? 1 : 0) + (z[1] > x ? 1 : 0);
                }
                const int fresh = min(16, rows_max(pc));
                for (int i = 0; i < fresh; i += 4) {
                    const u64x2 y = *reinterpret_cast<const u64x2*>(pe + i), z = *reinterpret_cast<const u64x2*>(pe + i + 2);
                    rx += (y[0] > x ? 1 : 0) + (y[1] > x ? 1 : 0) + (z[0] > x ? 1 : 0) + (z[1] > x ? 1 : 0);
                    rk += (y[0] > k ? 1 : 0) + (y[1] > k ? 1 : 0) + (z[0] > k ? 1 : 0) + (z[1] > k ? 1 : 0);
                }
                const u64 later = pe[16 + l];
                __builtin_amdgcn_wave_barrier();
                if (k && rk < n) kept[qr][rk] = k;
                if (x && rx < n) kept[qr][rx] = x;
                pe[l] = later;
                pe[16 + l] = 0ull;
                __builtin_amdgcn_wave_barrier();
                k = l < min(n, have + min(pc, 16)) ? kept[qr][l] : 0ull;
                if (have + min(pc, 16) >= n) bar = max(bar, kept[qr][n - 1]);
                pc = max(0, pc - 16);
                __builtin_amdgcn_wave_barrier();
            };
            for (int s0 = 0, span = steps; s0 < steps;) {
                const int s1 = min(steps, s0 + span);
                const float thr = bar ? key_score((unsigned)(bar >> 32)) : -INFINITY;      // later fours lose ties
                unsigned hit = 0;                                                 // four bits a step
                for (int i = s0, bit = 0; i < s1; ++i, bit += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(gp + i * 64);
                    hit |= ((x.x > thr ? 1u : 0u) | (x.y > thr ? 2u : 0u) | (x.z > thr ? 4u : 0u) | (x.w > thr ? 8u : 0u)) << bit;
                }
                const int cnt = __popc(hit);
                const int total = row_sum(cnt), most = rows_max(total);
                if (most > kGroupList && span > 1) { span = 1; continue; }       // many ties: 64 fours of a query at a time
                if (most > 0) {
                    int pos = cnt;                                                // sum over the lanes before
                    pos += __builtin_amdgcn_update_dpp(0, pos, 0x111, 0xf, 0xf, true);
                    pos += __builtin_amdgcn_update_dpp(0, pos, 0x112, 0xf, 0xf, true);
                    pos += __builtin_amdgcn_update_dpp(0, pos, 0x114, 0xf, 0xf, true);
                    pos += __builtin_amdgcn_update_dpp(0, pos, 0x118, 0xf, 0xf, true);
                    pos -= cnt;
                    while (__ballot(hit != 0)) {
                        if (hit) {
                            const int bit = __ffs((int)hit) - 1;
                            hit &= hit - 1;
                            fo[pos++] = (unsigned short)((s0 + (bit >> 2)) * 64 + l * 4 + (bit & 3));
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                    // sixteen scores of every query: LB lanes read one block's bounds together (16 bytes each, whole lines) and add up, lane e keeps score e
                    for (int r0 = 0; r0 < most; r0 += 4) {
                        const bool there = r0 + (l >> 2) < total;
                        const int j = there ? j0 + fo[r0 + (l >> 2)] * 4 + (l & 3) : NB;
                        float w = sp[min(j, NB - 1)], dot = 0.f;
                        w = j < last ? w : -1.0f;
                        f16x8 x[LB][CPL];
                        const unsigned end = (unsigned)(NB - 1) * (2 * D) + l % LB * 8;          // the last block's bounds
#pragma unroll
                        for (int f = 0; f < LB / 4; ++f) {
                            const unsigned at = (unsigned)(j0 + fo[min(r0 + l / LB * (LB / 4) + f, kGroupList - 1)] * 4) * (2 * D) + l % LB * 8;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
#pragma unroll
                                for (int c = 0; c < CPL; ++c) x[f * 4 + e][c] = *reinterpret_cast<const f16x8*>(kp + min(at + e * 2 * D, end) + c * LB * 8);
                        }
#pragma unroll
                        for (int e = 0; e < LB; ++e) {
                            float d = 0.f;
#pragma unroll
                            for (int c = 0; c < CPL; ++c)
#pragma unroll
                                for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_fdot2(h2{x[e][c][i], x[e][c][i + 1]}, h2{y[c][i], y[c][i + 1]}, d, false);      // whole numbers: exact
                            d += dpp_f<0xB1>(d);
                            d += dpp_f<0x4E>(d);
                            if constexpr (LB >= 8) d += dpp_f<0x141>(d);
                            if constexpr (LB >= 16) d += dpp_f<0x140>(d);
                            dot = l % LB == e ? d : dot;
                        }
                        const unsigned key = w < 0.f ? 0u : order_key(dot * w);
                        const u64 entry = key ? (u64)key << 32 | (unsigned)~j : 0ull;
                        const bool in = entry > bar;
                        const unsigned mine = (unsigned)(__ballot(in) >> (row * 16)) & 0xffffu;
                        if (in) pe[pc + __popc(mine & ((1u << l) - 1))] = entry;
                        pc += __popc(mine);
                        __builtin_amdgcn_wave_barrier();
                        while (rows_max(pc) > 16) flush();
                    }
                    while (rows_max(pc) > 0) flush();
                }
                s0 = s1;
            }
        }
        __syncthreads();
    }
    {
        const int t = t0 + qr;
        const u64 k = kept[qr][l];
        // in the order of the blocks: ~block is larger for the earlier ones
        const unsigned x = (unsigned)k;
        int rank = 0;
        each_ror<1, 16>([&](auto r) { rank += row_ror<decltype(r)::value>(x) > x ? 1 : 0; });
        __builtin_amdgcn_wave_barrier();
        pe[l] = 0ull;
        __builtin_amdgcn_wave_barrier();
        if (k) pe[rank] = k;
        __builtin_amdgcn_wave_barrier();
        const u64 e = pe[l];
        if (t >= T_ || l >= n) return;
        const size_t at = ((size_t)b * T_ + t) * KV + h;
        if constexpr (PARTS) part[(at * parts + blockIdx.x % parts) * n + l] = make_uint2((unsigned)(e >> 32), ~(unsigned)e);
        else out[at * n + l] = e ? (int)~(unsigned)e : -1;
    }
}

// the n best of the parts' n best: one wave per (query, kv head); the parts are in the order of the blocks
__global__ __launch_bounds__(64) void bs_select_join_kernel(const uint2* __restrict__ part, int parts, int n, int32_t* __restrict__ out) {
    __shared__ unsigned lk[64];
    __shared__ int li[64];
    constexpr int E = 4;
    const int lane = threadIdx.x, total = parts * n;
    const uint2* p = part + (size_t)blockIdx.x * total;
    unsigned key = 0u, least = 0u;
    int idx = -1, have = 0;
    for (int i0 = 0; i0 < total; i0 += E * 64) {
        unsigned c[E];
        int x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint2 v = i0 + e * 64 + lane < total ? p[i0 + e * 64 + lane] : make_uint2(0u, 0xffffffffu);
            c[e] = v.x;
            x[e] = (int)v.y;
        }
        take(key, idx, have, least, c, [&](int e) { return x[e]; }, n, lk, li, lane);
    }
    if (lane < n) out[(size_t)blockIdx.x * n + lane] = lane < have ? idx : -1;
}

// ------------------------------------------------------------------------------------------------------------ lists
// Counting sort of the mentions of a (sample, kv head) by block, in three launches: counts of `runs` runs of mentions, places, fill.  In the fill one wave
// takes a run (or a part of one) in order; equal blocks among its 64 lanes are found with one ballot per bit of the block number, counters live in LDS.  Same
// lists whatever the timing.  Bound by latency: 2.25 million mentions of 2200 blocks: count 7, places 8, scan 7, fill 37 us.
__device__ __forceinline__ int mention(const int32_t* blocks, unsigned e, unsigned e1, size_t bt0, int KV, int h, unsigned n, int& m) {
    if (e >= e1) return -1;
    const unsigned t = e / n, s = e - t * n;
    m = (int)(t * kMaxPick + s);
    return blocks[((bt0 + t) * KV + h) * n + s];
}

__global__ __launch_bounds__(256) void bs_count_kernel(const int32_t* __restrict__ blocks, int T_, int KV, int NB, int n, int runs, int run_len, int32_t* __restrict__ hist) {
    extern __shared__ int cnt[];
    const int run = blockIdx.x, bh = blockIdx.y, b = bh / KV, h = bh % KV;
    for (int j = threadIdx.x; j < NB; j += 256) cnt[j] = 0;
    __syncthreads();
    const unsigned total = (unsigned)T_ * n, e0 = min(total, (unsigned)run * run_len), e1 = min(total, e0 + run_len);
    for (unsigned e = e0 + threadIdx.x; e < e1; e += 1024) {
        int j[4], m;
#pragma unroll
        for (int u = 0; u < 4; ++u) j[u] = mention(blocks, e + u * 256, e1, (size_t)b * T_, KV, h, n, m);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j[u] >= 0 && j[u] < NB) atomicAdd(&cnt[j[u]], 1);          // a count: any order
    }
    __syncthreads();
    int32_t* hp = hist + ((size_t)bh * runs + run) * NB;
    for (int j = threadIdx.x; j < NB; j += 256) hp[j] = cnt[j];
}

// W waves share a run (a part each, in order): a step of 64 mentions is one chain of dependent instructions, about 3000 cycles, so the time is the steps of a
// wave; more runs would do as well, but each costs counters in memory.  Four waves where their counters fit in 64 KB of LDS, else one.
template <int W>
__global__ __launch_bounds__(W * 64) void bs_fill_kernel(const int32_t* __restrict__ blocks, int T_, int KV, int NB, int n, int runs, int run_len, int bits,
                                                         const int32_t* __restrict__ hist, const int32_t* __restrict__ start, int32_t* __restrict__ list) {
    extern __shared__ int counters[];                    // [W][NB]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, run = blockIdx.x, bh = blockIdx.y, b = bh / KV, h = bh % KV;
    const unsigned total = (unsigned)T_ * n, first = min(total, (unsigned)run * run_len), last = min(total, first + run_len);
    const unsigned part = (run_len / 64 + W - 1) / W * 64, e0 = min(last, first + wave * part), e1 = min(last, e0 + part);
    int* cnt = counters + wave * NB;
    constexpr int U = 4;
    int j[U], m[U];
    if constexpr (W > 1) {
        for (int i = threadIdx.x; i < W * NB; i += W * 64) counters[i] = 0;
        __syncthreads();
        for (unsigned e = e0; e < e1; e += U * 64) {
#pragma unroll
            for (int u = 0; u < U; ++u) j[u] = mention(blocks, e + u * 64 + lane, e1, (size_t)b * T_, KV, h, n, m[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j[u] >= 0 && j[u] < NB) atomicAdd(&cnt[j[u]], 1);      // a count: any order
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) j[u] = mention(blocks, e0 + u * 64 + lane, e1, (size_t)b * T_, KV, h, n, m[u]);
    const int32_t *hp = hist + ((size_t)bh * runs + run) * NB, *sp = start + (size_t)bh * (NB + 1);
    for (int j0 = threadIdx.x; j0 < NB; j0 += 4 * W * 64) {
        int x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = j0 + i * W * 64;
            x[i] = at < NB ? hp[at] + sp[at] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = j0 + i * W * 64;
            if (at >= NB) break;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int c = W > 1 ? counters[w * NB + at] : 0;
                counters[w * NB + at] = x[i];
                x[i] += c;
            }
        }
    }
    __syncthreads();
    for (unsigned e = e0; e < e1; e += U * 64) {
        int jn[U], mn[U];                                                  // the next mentions are on their way
#pragma unroll
        for (int u = 0; u < U; ++u) jn[u] = mention(blocks, e + (U + u) * 64 + lane, e1, (size_t)b * T_, KV, h, n, mn[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ok = j[u] >= 0 && j[u] < NB;
            unsigned long long same = __ballot(ok);
            for (int bit = 0; bit < bits; ++bit) {
                const unsigned long long x = __ballot(ok && (j[u] >> bit & 1));
                same &= (j[u] >> bit & 1) ? x : ~x;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const int at = ok ? cnt[j[u]] + rank : 0;
            __builtin_amdgcn_wave_barrier();
            if (ok && rank == 0) cnt[j[u]] += __popcll(same);
            __builtin_amdgcn_wave_barrier();
            if (ok) list[(size_t)bh * total + at] = m[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) { j[u] = jn[u]; m[u] = mn[u]; }
    }
}

// counts of the runs -> places within a block's list, and its length.  64 blocks a workgroup, 16 threads a block with a stretch of the runs each
__global__ __launch_bounds__(1024) void bs_places_kernel(int32_t* __restrict__ hist, int runs, int NB, int32_t* __restrict__ len) {
    __shared__ int sums[16][64];
    const int c = threadIdx.x & 63, part = threadIdx.x >> 6, j = blockIdx.x * 64 + c, bh = blockIdx.y;
    const int per = (runs + 15) / 16, r0 = min(runs, part * per), r1 = min(runs, r0 + per);
    int32_t* hp = hist + (size_t)bh * runs * NB + j;
    int sum = 0;
    if (j < NB) {
#pragma unroll 8
        for (int r = r0; r < r1; ++r) sum += hp[(size_t)r * NB];
    }
    sums[part][c] = sum;
    __syncthreads();
    if (j >= NB) return;
    int at = 0;
    for (int p = 0; p < part; ++p) at += sums[p][c];
    if (part == 15) len[(size_t)bh * (NB + 1) + j] = at + sum;
    for (int r = r0; r < r1; r += 8) {
        int x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r + i < r1 ? hp[(size_t)(r + i) * NB] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r + i < r1) {
                hp[(size_t)(r + i) * NB] = at;
                at += x[i];
            }
    }
}

// one workgroup per (sample, kv head): lengths -> starts of the lists (in place), work items of at most `rows` rows
__global__ __launch_bounds__(1024) void bs_scan_kernel(int NB, int G, int rows, int max_items, int32_t* __restrict__ start, int32_t* __restrict__ items,
                                                       int32_t* __restrict__ n_items) {
    __shared__ int ws[2][16];
    __shared__ int carry[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bh = blockIdx.x;
    if (tid < 2) carry[tid] = 0;
    __syncthreads();
    for (int j0 = 0; j0 < NB; j0 += 1024) {
        const int j = j0 + tid;
        const int len = j < NB ? start[(size_t)bh * (NB + 1) + j] : 0;
        const int its = (int)(((long long)len * G + rows - 1) / rows);
        int a = len, c = its;          // inclusive scans over the workgroup
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(a, o), y = __shfl_up(c, o);
            if (lane >= o) { a += x; c += y; }
        }
        if (lane == 63) { ws[0][wave] = a; ws[1][wave] = c; }
        __syncthreads();
        int pa = carry[0], pc = carry[1];
        for (int w = 0; w < wave; ++w) { pa += ws[0][w]; pc += ws[1][w]; }
        if (j < NB) {
            start[(size_t)bh * (NB + 1) + j] = pa + a - len;
            for (int i = 0; i < its; ++i) {
                int32_t* it = items + ((size_t)bh * max_items + pc + c - its + i) * 2;
                it[0] = j;
                it[1] = i * rows;
            }
        }
        __syncthreads();
        if (tid == 1023) { carry[0] = pa + a; carry[1] = pc + c; }
        __syncthreads();
    }
    if (tid == 0) { start[(size_t)bh * (NB + 1) + NB] = carry[0]; n_items[bh] = carry[1]; }
}

// ------------------------------------------------------------------------------------------------------------ tiles
// Operands of the 32 x 32 x 16 matrix instructions: a lane holds eight consecutive k of its row; a contraction over d walks d = 16 s + 8 half + i.
// Accumulators: column lane & 31, rows 8 (i / 4) + 4 half + i % 4; a contraction over keys or queries takes such a tile as the B operand as it lies: step s
// of 16 covers rows 16 s + 4 half + {0..3, 8..11}.
//
// fp32 tensors run on the fp32 instruction, 32 x 32 x 2: the eight elements of a piece one after the other, so that nothing of a value's 24 bits or of its range is
// lost beside another one (an infinity among the values stays one).  Two fp16 terms of values relative to the largest of their block are faster (281600 queries x 8 blocks:
// forward 206 us against 285, backward 597 against 814) and hold 22 bits, but only of values within 2^-18 of that largest: one huge value took the others' bits.
template <typename T> struct Op;
template <> struct Op<__bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Op<_Float16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Op<float> {
    typedef float frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};
template <typename T> constexpr bool kNarrow = std::is_same<T, _Float16>::value;      // P and dS need a common power of two

template <typename T, int D> struct Shape {
    static constexpr int KS = D / 16;                           // k-steps over d
    static constexpr int DT = (D + 31) / 32;                    // 32-wide tiles of d
    static constexpr int P = D + 16 / (int)sizeof(T);           // row pitch of a [row][d] tile: banks
    static constexpr int PT = kKeys + 4;                        // row pitch of a [d][key] tile
    static constexpr int kRowTile = kKeys * P;
    static constexpr int kTransTile = DT * 32 * PT;             // d padded to 32 with zeros
};

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// eight elements on a 16-byte address, in pieces of 16 bytes
template <typename T> __device__ __forceinline__ typename tok_vec<T>::v8 get8(const T* p) {
    if constexpr (is_f32<T>::value) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *reinterpret_cast<const typename tok_vec<T>::v8*>(p);
    }
}
template <typename T> __device__ __forceinline__ void put8(T* p, typename tok_vec<T>::v8 x) {
    if constexpr (is_f32<T>::value) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *reinterpret_cast<typename tok_vec<T>::v8*>(p) = x;
    }
}

// the power of two that brings m to 2^14 .. 2^15, the top of fp16: values down to 2^-18 of the largest keep 22 bits in two terms, and what is below that is off by
// 2^-39 of it at most (half of fp16's last step, 2^-25, beside 2^14)
__device__ __forceinline__ float pow2_over(float m) {
    return m < INFINITY ? ldexpf(1.0f, max(__builtin_amdgcn_frexp_expf(m) - 15, -126)) : 1.0f;      // (its reciprocal stays finite)
}

// rows [0, 64) of a block to LDS: [key][d], and [d][key] of DA channels from d0 on.  Keys behind the end or masked are zeros.
// All 256 threads; ends with the writes, not with a barrier.
template <typename T, int D, bool ROW, bool TRANS, int DA = D>
__device__ __forceinline__ void load_block(const T* src, long long st, int t0, unsigned long long seen, T* row, T* tr, int d0 = 0) {
    using S = Shape<T, D>;
    constexpr int CPR = D / 8, N = kKeys * CPR / 256 > 0 ? kKeys * CPR / 256 : 1;
    typedef typename tok_vec<T>::v8 vec;
    vec x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = threadIdx.x + u * 256, key = i & 63, c = i >> 6;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][e] = (T)0.f;
        if (c < CPR && (seen >> key & 1)) x[u] = get8(src + (long long)(t0 + key) * st + c * 8);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = threadIdx.x + u * 256, key = i & 63, c = i >> 6;
        if (c >= CPR) continue;
        if constexpr (ROW) put8(row + key * S::P + c * 8, x[u]);
        if constexpr (TRANS) {
            const int d = c * 8 - d0;
            if (DA == D || (d >= 0 && d < DA)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) tr[(d + e) * S::PT + key] = x[u][e];
            }
        }
    }
    if constexpr (TRANS && D < 32) {
        for (int i = threadIdx.x; i < (32 - D) * S::PT; i += 256) tr[D * S::PT + i] = (T)0.f;
    }
}

// a head vector in pieces of one k-step, straight from global memory; the two half waves hold halves of it
template <typename T, int D> struct RowFrags { typename Op<T>::frag f[D / 16]; };
template <typename T, int D> __device__ __forceinline__ RowFrags<T, D> load_row(const T* p, bool in, int half) {
    RowFrags<T, D> r;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.f[s][e] = (T)0.f;
        if (in) r.f[s] = get8(p + s * 16 + half * 8);
    }
    return r;
}

// acc += (32 rows of an LDS tile) x (32 row vectors in registers), over d; SWAP: the LDS rows are the columns of the result
template <typename T, int D, bool SWAP>
__device__ __forceinline__ f32x16 mma_d(const T* tile, int r, int half, const RowFrags<T, D>& q, f32x16 acc) {
    using S = Shape<T, D>;
#pragma unroll
    for (int s = 0; s < S::KS; ++s) {
        const typename Op<T>::frag x = get8(tile + r * S::P + s * 16 + half * 8);
        acc = SWAP ? Op<T>::mma(q.f[s], x, acc) : Op<T>::mma(x, q.f[s], acc);
    }
    return acc;
}

// A 32 x 32 tile of P or dS as B operand: fp32 as it is, for 16-bit tensors in two terms -- the product then has the precision of fp32 probabilities and the result's own
// rounding is the only one that counts.  RANGE: the backward's tiles have no largest value to be relative to, and fp16 ends at 2^-24: a column (a lane and the one 32
// further, in the operand and in the result) is brought to the top of its range by a power of two, and the product brought back (gradients of a scaled or a small loss
// keep their precision); bf16 has the range.  The first fp16 term is cut, not rounded (one instruction for two): the second, rounded, holds what it leaves.
template <typename T, bool RANGE> struct Split {
    static constexpr bool two = !is_f32<T>::value, far = RANGE && kNarrow<T>;
    typename Op<T>::frag hi[2], lo[2];
    float back = 1.0f;
    __device__ __forceinline__ explicit Split(const f32x16& p) {
        float to = 1.0f;
        if constexpr (far) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(p[i]));
            m = fmaxf(m, __shfl_xor(m, 32));
            back = pow2_over(m);
            to = 1.0f / back;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float x = far ? p[s * 8 + e] * to : p[s * 8 + e], y = far ? p[s * 8 + e + 1] * to : p[s * 8 + e + 1];
                T h, g;
                if constexpr (kNarrow<T>) {
                    const auto c = __builtin_amdgcn_cvt_pkrtz(x, y);
                    h = (T)c[0];
                    g = (T)c[1];
                } else {
                    h = (T)x;
                    g = (T)y;
                }
                hi[s][e] = h;
                hi[s][e + 1] = g;
                if constexpr (two) {
                    lo[s][e] = (T)(x - (float)h);
                    lo[s][e + 1] = (T)(y - (float)g);
                }
            }
    }
};

// acc (d x columns) += A^T (d x 32 rows) p (32 rows x columns): A in LDS as [d][row]
template <typename T, bool RANGE>
__device__ __forceinline__ f32x16 mma_rows(const T* a, int pitch, int lane, const Split<T, RANGE>& x, f32x16 acc) {
    typedef typename tok_vec<T>::v4 v4;
    const int half = lane >> 5, m = lane & 31;
    constexpr bool far = Split<T, RANGE>::far;
    f32x16 t = far ? zero16() : acc;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const v4 u = *reinterpret_cast<const v4*>(a + m * pitch + s * 16 + half * 4), w = *reinterpret_cast<const v4*>(a + m * pitch + s * 16 + half * 4 + 8);
        const typename Op<T>::frag f = __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (Split<T, RANGE>::two) t = Op<T>::mma(f, x.lo[s], t);
        t = Op<T>::mma(f, x.hi[s], t);
    }
    if constexpr (far) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] += t[i] * x.back;
        return acc;
    }
    return t;
}

__device__ __forceinline__ unsigned long long seen_keys(const BsArgs& a, int b, int j) {       // visible keys of a block, same in every lane
    const int t = j * kKeys + (threadIdx.x & 63);
    return __ballot(t < a.Nk && (!a.mask || a.mask[(size_t)b * a.Nk + t]));
}

// scores of keys that are not visible: -inf (rows of a tile of keys x queries)
__device__ __forceinline__ void hide(f32x16& s, unsigned long long seen, int kt, int half) {
    const unsigned bits = (unsigned)(seen >> (kt * 32)) >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = bits >> (8 * (i / 4) + (i & 3)) & 1 ? s[i] : -INFINITY;
}

// the mention a row stands for: row = mention * G + head of the group
struct Row { bool in; int t, slot, head; };
__device__ __forceinline__ Row row_of(const BsArgs& a, const int32_t* list, int len, int h, int r) {
    Row x;
    const int e = a.G == 1 ? r : (int)((unsigned)r / (unsigned)a.G);
    x.in = e < len;
    const int m = x.in ? list[e] : 0;
    x.t = m / kMaxPick;
    x.slot = m % kMaxPick;
    x.head = h * a.G + (a.G == 1 ? 0 : r - e * a.G);
    return x;
}

// Rows (mentions x heads of the group) of a work item: 1024, which reads K and V once for all queries of a block of average fame, down to 512 where that leaves fewer
// than 1024 items.  Measured (us, forward / with backward, items of 512 | 1024 | 2048): 35200 x 35200, 8 heads of 32, 8 blocks, fp32: 369 / 1230 | 379 / 1249 | 403 / 1319
// (512 gains 2 % there, at twice the slabs in the workspace); 4400 x 8789, 4 of 64, bf16: 53 / 152 | 61 / 167 | 77 / 210; 600 x 35189, 8 of 64 over 2, 16 blocks:
// 49 / 136 | 56 / 155 | 69 / 180; 256 or 128 there cost the backward more slabs than they bring (4400: 164, 189 where 512 took 158).
constexpr int kItemRows = 1024, kItemLeast = 512;

// ------------------------------------------------------------------------------------------------------------ attention, many queries
// A mention's record: (maximum (scaled, base 2), sum) and the attention over its block alone, next to each other -- they are written to places all over the
// workspace, and 8 bytes of their own would cost a memory request as large as the rest.  All in fp32 whatever the tensors' type: the output is rounded once, and is the
// same with and without gradients (held in 16 bits the records halve the bytes of the join, at 1.4 times the error of the output's own rounding).
template <int D> struct Record {
    static constexpr size_t bytes = 8 + D * 4;
    static __device__ __forceinline__ char* at(void* part, size_t i) { return static_cast<char*>(part) + i * bytes; }
    static __device__ __forceinline__ const char* at(const void* part, size_t i) { return static_cast<const char*>(part) + i * bytes; }
    typedef f32x4 v4 __attribute__((aligned(8)));
    static __device__ __forceinline__ void put(char* r, int d, f32x4 v) { *reinterpret_cast<v4*>(r + 8 + d * 4) = v; }
    static __device__ __forceinline__ f32x4 get(const char* r, int d) { return *reinterpret_cast<const v4*>(r + 8 + d * 4); }
};

// 281600 queries x 8 blocks of 32 channels: bf16 197 us, fp32 285 us.  fp32: the matrix cores are busy in 52 % of the cycles (120 us of products at their measured rate),
// vector instructions issue in 21 %.  bf16: 7 % and 41 %, and a wave waits 60 % of its time, mostly for memory: the records go to places all over the workspace, 306 MB
// (62 us at the rate of a large copy) as pieces of two or three cache lines each.  The launch bounds keep one more wave on a SIMD than the compiler would (whole call,
// 17600 queries x 4 heads of 64 fp32: 207 us against 246, 8800 x 4 of 128 bf16: 105 against 116).
template <typename T, int D>
__global__ __launch_bounds__(256, (is_f32<T>::value ? (D <= 32 ? 3 : D == 64 ? 2 : 1) : (D <= 32 ? 4 : D == 64 ? 3 : 2))) void bs_forward_kernel(BsArgs a) {
    using S = Shape<T, D>;
    __shared__ __align__(16) T lk[S::kRowTile];
    __shared__ __align__(16) T lv[S::kTransTile];
    const int bh = blockIdx.y, b = bh / a.KV, h = bh % a.KV;
    if ((int)blockIdx.x >= a.n_items[bh]) return;
    const int32_t* it = a.items + ((size_t)bh * a.max_items + blockIdx.x) * 2;
    const int j = it[0], first = it[1];
    const int32_t* st = a.start + (size_t)bh * (a.NB + 1) + j;
    const int len = st[1] - st[0];
    const int32_t* list = a.list + (size_t)bh * a.T * a.n + st[0];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int last = min(first + a.item_rows, len * a.G);
    const T* qbase = static_cast<const T*>(a.q) + b * a.qb;
    // the first queries are on their way before K and V, the next ones during the work on these
    Row r = row_of(a, list, len, h, first + wave * 32 + (lane & 31));
    RowFrags<T, D> raw = load_row<T, D>(qbase + r.t * a.qt + r.head * a.qh, r.in, half);
    const unsigned long long seen = seen_keys(a, b, j);
    load_block<T, D, true, false>(static_cast<const T*>(a.k) + b * a.kb + h * a.kh, a.kt, j * kKeys, seen, lk, nullptr);
    load_block<T, D, false, true>(static_cast<const T*>(a.v) + b * a.vb + h * a.vh, a.vt, j * kKeys, seen, nullptr, lv);
    __syncthreads();
    const float c = a.scale * kLog2e;
    Row ahead = row_of(a, list, len, h, first + wave * 32 + 128 + (lane & 31));
    for (int r0 = first + wave * 32; r0 < last; r0 += 128) {
        const RowFrags<T, D> qf = raw;
        const Row next = ahead;
        if (r0 + 128 < last) {
            raw = load_row<T, D>(qbase + next.t * a.qt + next.head * a.qh, next.in, half);
            ahead = row_of(a, list, len, h, r0 + 256 + (lane & 31));
        }
        f32x16 s[2];
        float m = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            s[kt] = mma_d<T, D, false>(lk, kt * 32 + (lane & 31), half, qf, zero16());
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kt][i] *= c;
            if (seen != ~0ull) hide(s[kt], seen, kt, half);
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, s[kt][i]);
        }
        m = fmaxf(m, __shfl_xor(m, 32));
        constexpr float kTop = kNarrow<T> ? 15.f : 0.f;               // fp16 terms: from the top of their range as well
        const float base = m == -INFINITY ? 0.f : m - kTop;
        float l = 0.f;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kt][i] = __builtin_amdgcn_exp2f(s[kt][i] - base);
                l += s[kt][i];
            }
        l += __shfl_xor(l, 32);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if constexpr (kNarrow<T>) l *= 1.0f / 32768.f;
        char* rec = Record<D>::at(a.part, (((size_t)b * a.T + r.t) * a.H + r.head) * a.n + r.slot);
        const Split<T, false> p0(s[0]), p1(s[1]);
#pragma unroll
        for (int dt = 0; dt < S::DT; ++dt) {
            f32x16 o = mma_rows<T>(lv + dt * 32 * S::PT, S::PT, lane, p0, zero16());
            o = mma_rows<T>(lv + dt * 32 * S::PT + 32, S::PT, lane, p1, o);
            if (r.in) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = dt * 32 + 8 * i + 4 * half;
                    if (d < D) Record<D>::put(rec, d, f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]} * inv);
                }
            }
        }
        if (r.in && half == 0) *reinterpret_cast<f32x2*>(rec) = f32x2{m, l};
        r = next;
    }
}

// ------------------------------------------------------------------------------------------------------------ attention, few queries
// One wave per mention, all heads of its group: a lane per key for the scores, D / 8 lanes per key for the values.  Bound by the latency of two rounds of loads
// (one query x 8 heads x 16 blocks: 5.5 us).
template <typename T, int D>
__global__ __launch_bounds__(64) void bs_few_kernel(BsArgs a) {
    __shared__ __align__(16) float lq[D];
    __shared__ float lp[kKeys];
    const int lane = threadIdx.x;
    const long long w = blockIdx.x;                      // (b, t, kv head, slot)
    const int slot = (int)(w % a.n), h = (int)(w / a.n % a.KV);
    const long long bt = w / a.n / a.KV;
    const int b = (int)(bt / a.T), t = (int)(bt - (long long)b * a.T);
    const int j = a.blocks[w];
    if (j < 0 || j >= a.NB) return;
    const unsigned long long seen = seen_keys(a, b, j);
    const bool mine = seen >> lane & 1;
    const T* kp = static_cast<const T*>(a.k) + b * a.kb + h * a.kh + (long long)(j * kKeys + (mine ? lane : 0)) * a.kt;
    constexpr int LPK = D / 8, KPS = 64 / LPK;
    const int sub = lane % LPK, kq = lane / LPK;
    const T* vp = static_cast<const T*>(a.v) + b * a.vb + h * a.vh + (long long)j * kKeys * a.vt + sub * 8;
    for (int g = 0; g < a.G; ++g) {
        const T* qp = static_cast<const T*>(a.q) + b * a.qb + (long long)t * a.qt + (long long)(h * a.G + g) * a.qh;
        __syncthreads();
        for (int d = lane; d < D; d += 64) lq[d] = (float)qp[d];
        __syncthreads();
        float s = -INFINITY;
        if (mine) {
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < D; d += 4) acc += tok_load4(kp + d) * *reinterpret_cast<const f32x4*>(lq + d);
            s = ((acc.x + acc.y) + (acc.z + acc.w)) * (a.scale * kLog2e);
        }
        float m = s;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float p = __builtin_amdgcn_exp2f(s - (m == -INFINITY ? 0.f : m));
        float l = p;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
        lp[lane] = p;
        __syncthreads();
        f32x4 o0{0.f, 0.f, 0.f, 0.f}, o1 = o0;
#pragma unroll
        for (int i = 0; i < kKeys / KPS; ++i) {
            const int key = i * KPS + kq;
            if (seen >> key & 1) {
                const float x = lp[key];
                o0 += tok_load4(vp + (long long)key * a.vt) * x;
                o1 += tok_load4(vp + (long long)key * a.vt + 4) * x;
            }
        }
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) { o0[e] += __shfl_xor(o0[e], o); o1[e] += __shfl_xor(o1[e], o); }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        char* rec = Record<D>::at(a.part, (((size_t)b * a.T + t) * a.H + h * a.G + g) * a.n + slot);
        if (lane < LPK) {
            Record<D>::put(rec, sub * 8, o0 * inv);
            Record<D>::put(rec, sub * 8 + 4, o1 * inv);
        }
        if (lane == 0) *reinterpret_cast<f32x2*>(rec) = f32x2{m, l};
    }
}

// The n places of a query joined: D / 4 lanes a (query, head).  Bound by HBM (281600 x 8 records of 136 bytes: 73 us, 4.4 TB/s).  rest: what the output's rounding took away, for the backward's sum dO O
template <typename T, int D>
__global__ __launch_bounds__(256) void bs_join_kernel(BsArgs a, long long rows) {
    constexpr int L = D / 4;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int sub = threadIdx.x % L;
    if (r >= rows) return;
    const unsigned hq = (unsigned)(r % a.H);
    const long long bt = r / a.H;
    const int32_t* bl = a.blocks + (bt * a.KV + hq / (unsigned)a.G) * a.n;
    const char* part = Record<D>::at(a.part, (size_t)(r * a.n));
    float m = -INFINITY, l = 0.f;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.n; s0 += 8) {                // eight places at a time, all their loads in flight
        f32x2 x[8];
        f32x4 y[8];
        float mm = m;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = s0 + u, j = s < a.n ? bl[s] : -1;
            const bool ok = j >= 0 && j < a.NB;          // other places were never written
            x[u] = f32x2{-INFINITY, 0.f};
            y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (ok) {
                const char* rec = part + (size_t)s * Record<D>::bytes;
                x[u] = *reinterpret_cast<const f32x2*>(rec);
                y[u] = Record<D>::get(rec, sub * 4);
            }
            mm = fmaxf(mm, x[u].x);
        }
        const float base = mm == -INFINITY ? 0.f : mm, f = __builtin_amdgcn_exp2f(m - base);
        l *= f;
        o *= f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = __builtin_amdgcn_exp2f(x[u].x - base) * x[u].y;
            l += w;
            o += y[u] * w;
        }
        m = mm;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    o *= inv;
    tok_store4(static_cast<T*>(a.out) + r * D + sub * 4, o);
    if (a.rest) {
        typedef typename tok_vec<T>::v4 v4;
        tok_store4(static_cast<T*>(a.rest) + r * D + sub * 4, o - __builtin_convertvector(__builtin_convertvector(o, v4), f32x4));
    }
    if (a.lse && sub == 0) a.lse[r] = l == 0.f ? INFINITY : m + log2f(l);
}

// ------------------------------------------------------------------------------------------------------------ backward
// (log-sum-exp, sum dO O) of every (query, head), next to each other: a mention reads both at once
template <typename T, int D>
__global__ __launch_bounds__(256) void bs_delta_kernel(const T* __restrict__ out, const T* __restrict__ rest, const T* __restrict__ dout, const float* __restrict__ lse, f32x2* __restrict__ ld,
                                                       long long rows) {
    constexpr int L = D / 4;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int sub = threadIdx.x % L;
    if (r >= rows) return;
    f32x4 o = tok_load4(out + r * D + sub * 4);
    if (rest) o += tok_load4(rest + r * D + sub * 4);
    const f32x4 p = o * tok_load4(dout + r * D + sub * 4);
    float s = (p.x + p.y) + (p.z + p.w);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o);
    if (sub == 0) ld[r] = f32x2{lse[r], s};
}

// One workgroup per work item, four waves of 32 rows.  P and dP are computed twice, as keys x queries for dQ (a lane keeps a query) and as queries x
// keys for dK, dV (a lane keeps a key): two more products instead of a transpose through LDS.  DA: the part of d whose dK, dV, dQ this workgroup
// keeps (blockIdx.z-th).
// 281600 queries x 8 blocks of 32 channels, fp32: 814 us; seven products, 64.6 GFLOP, 420 us at the matrix cores' measured rate: they are busy in 62 % of the cycles, vector
// instructions issue in 14 %, at two waves a SIMD (205 registers of 256).  17600 x 8 of 64, bf16: 76 us; one wave a SIMD (registers and LDS), which waits for loads and
// LDS half of its time: matrix cores 8 %, vector issue 22 %.
template <typename T, int D, int DA>
__global__ __launch_bounds__(256, (D <= 32 ? 2 : 1)) void bs_backward_kernel(BsArgs a) {
    using S = Shape<T, D>;
    constexpr int AT = (DA + 31) / 32;                                     // d tiles of this workgroup
    constexpr int QP = 32 + 4, kWaveTile = AT * 32 * QP;                   // per-wave tile of 32 rows: [d][row]
    constexpr int kTrans = Shape<T, DA>::kTransTile;
    constexpr size_t kTiles = sizeof(T) * (2 * S::kRowTile + kTrans + 8 * kWaveTile);
    __shared__ __align__(16) char smem[kTiles > 32768 ? kTiles : 32768];   // the last sums take 32 KB
    T* lk = reinterpret_cast<T*>(smem);
    T* lv = lk + S::kRowTile;
    T* lkt = lv + S::kRowTile;
    T* lqs = lkt + kTrans;
    __shared__ __align__(16) f32x2 lld[4][32];
    const int bh = blockIdx.y, b = bh / a.KV, h = bh % a.KV, d0 = blockIdx.z * DA;
    if ((int)blockIdx.x >= a.n_items[bh]) return;
    const int32_t* it = a.items + ((size_t)bh * a.max_items + blockIdx.x) * 2;
    const int j = it[0], first = it[1];
    const int32_t* st = a.start + (size_t)bh * (a.NB + 1) + j;
    const int len = st[1] - st[0];
    const int32_t* list = a.list + (size_t)bh * a.T * a.n + st[0];
    const unsigned long long seen = seen_keys(a, b, j);
    load_block<T, D, true, true, DA>(static_cast<const T*>(a.k) + b * a.kb + h * a.kh, a.kt, j * kKeys, seen, lk, lkt, d0);
    load_block<T, D, true, false>(static_cast<const T*>(a.v) + b * a.vb + h * a.vh, a.vt, j * kKeys, seen, lv, nullptr);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    T* lq = lqs + wave * 2 * kWaveTile;
    T* lo = lq + kWaveTile;
    if constexpr (DA < 32) {                                               // channels behind D: zeros, once
        for (int i = lane; i < (32 - DA) * QP; i += 64) lq[DA * QP + i] = lo[DA * QP + i] = (T)0.f;
    }
    __syncthreads();
    const int last = min(first + a.item_rows, len * a.G);
    const float c = a.scale * kLog2e;
    f32x16 dk[AT][2], dv[AT][2];
#pragma unroll
    for (int t = 0; t < AT; ++t) { dk[t][0] = zero16(); dk[t][1] = zero16(); dv[t][0] = zero16(); dv[t][1] = zero16(); }
    Row ahead = row_of(a, list, len, h, first + wave * 32 + (lane & 31));
    for (int r0 = first + wave * 32; r0 < last; r0 += 128) {
        const Row r = ahead;
        const size_t qrow = ((size_t)b * a.T + r.t) * a.H + r.head;
        const RowFrags<T, D> qf = load_row<T, D>(static_cast<const T*>(a.q) + b * a.qb + r.t * a.qt + r.head * a.qh, r.in, half);
        const RowFrags<T, D> of = load_row<T, D>(static_cast<const T*>(a.dout) + qrow * D, r.in, half);
        const f32x2 ld = r.in ? a.ld[qrow] : f32x2{INFINITY, 0.f};         // rows that are not there: P = 0
        ahead = row_of(a, list, len, h, r0 + 128 + (lane & 31));
        if (half == 0) lld[wave][lane & 31] = ld;
#pragma unroll
        for (int s = 0; s < S::KS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = s * 16 + half * 8 + e - d0;
                if (DA == D || (d >= 0 && d < DA)) {
                    lq[d * QP + (lane & 31)] = qf.f[s][e];
                    lo[d * QP + (lane & 31)] = of.f[s][e];
                }
            }
        __builtin_amdgcn_wave_barrier();
        f32x16 dq[AT];
#pragma unroll
        for (int t = 0; t < AT; ++t) dq[t] = zero16();
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            // keys x queries
            f32x16 s = mma_d<T, D, false>(lk, kt * 32 + (lane & 31), half, qf, zero16()), p = mma_d<T, D, false>(lv, kt * 32 + (lane & 31), half, of, zero16());
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], c, -ld.x);
            if (seen != ~0ull) hide(s, seen, kt, half);
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(s[i]) * (p[i] - ld.y);
            {
                const Split<T, true> ds(p);
#pragma unroll
                for (int t = 0; t < AT; ++t) dq[t] = mma_rows<T>(lkt + t * 32 * S::PT + kt * 32, S::PT, lane, ds, dq[t]);
            }
            __builtin_amdgcn_sched_barrier(0);                             // one part's registers at a time
            // queries x keys
            s = mma_d<T, D, true>(lk, kt * 32 + (lane & 31), half, qf, zero16());
            p = mma_d<T, D, true>(lv, kt * 32 + (lane & 31), half, of, zero16());
            // (keys that are not visible: their columns are left out at the end)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const f32x2 x = lld[wave][8 * (i / 4) + 4 * half + (i & 3)];
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -x[0]));
                p[i] = s[i] * (p[i] - x[1]);
            }
            {
                const Split<T, true> rp(s);
#pragma unroll
                for (int t = 0; t < AT; ++t) dv[t][kt] = mma_rows<T>(lo + t * 32 * QP, QP, lane, rp, dv[t][kt]);
            }
            __builtin_amdgcn_sched_barrier(0);
            {
                const Split<T, true> rs(p);
#pragma unroll
                for (int t = 0; t < AT; ++t) dk[t][kt] = mma_rows<T>(lq + t * 32 * QP, QP, lane, rs, dk[t][kt]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_wave_barrier();
        if (r.in) {
            float* dst = static_cast<float*>(a.part) + (qrow * a.n + r.slot) * D + d0;
#pragma unroll
            for (int t = 0; t < AT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = t * 32 + 8 * i + 4 * half;
                    if (d < DA) *reinterpret_cast<f32x4*>(dst + d) = f32x4{dq[t][4 * i], dq[t][4 * i + 1], dq[t][4 * i + 2], dq[t][4 * i + 3]} * a.scale;
                }
        }
    }
    // the four waves' sums, in order, through LDS; a block with one work item is done here, others leave a slab
    float* red = reinterpret_cast<float*>(smem);
    const bool whole = len * a.G <= a.item_rows;
    float* slab = a.slab + ((size_t)bh * a.max_items + blockIdx.x) * 2 * kKeys * D;
#pragma unroll
    for (int w2 = 0; w2 < 2; ++w2)
#pragma unroll
        for (int t = 0; t < AT; ++t) {
            __syncthreads();
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const f32x16& x = w2 ? dv[t][kt] : dk[t][kt];
                    *reinterpret_cast<f32x4*>(red + (((wave * 2 + kt) * 4 + i / 4) * 64 + lane) * 4) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
                }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = threadIdx.x + u * 256, ln = i & 63, i4 = i >> 6 & 3, kt = i >> 8;
                f32x4 y = *reinterpret_cast<const f32x4*>(red + i * 4);
#pragma unroll
                for (int w = 1; w < 4; ++w) y += *reinterpret_cast<const f32x4*>(red + (w * 512 + i) * 4);
                const int key = kt * 32 + (ln & 31), d = t * 32 + 8 * i4 + 4 * (ln >> 5), tok = j * kKeys + key;
                if (d >= DA) continue;
                y = seen >> key & 1 ? y * (w2 ? 1.0f : a.scale) : f32x4{0.f, 0.f, 0.f, 0.f};
                if (whole) {
                    T* dst = static_cast<T*>(w2 ? a.dv : a.dk);
                    if (dst && tok < a.Nk) tok_store4(dst + (((size_t)b * a.Nk + tok) * a.KV + h) * D + d0 + d, y);
                } else {
                    *reinterpret_cast<f32x4*>(slab + ((size_t)w2 * kKeys + key) * D + d0 + d) = y;
                }
            }
        }
}

// dK, dV of the blocks that nobody named (zeros) or that took several work items: their slabs, in order.  One workgroup per (block, sample, kv head).
template <typename T, int D>
__global__ __launch_bounds__(256) void bs_dkv_kernel(BsArgs a) {
    const int j = blockIdx.x, bh = blockIdx.y, b = bh / a.KV, h = bh % a.KV;
    const int32_t* st = a.start + (size_t)bh * (a.NB + 1) + j;
    const int rows = (st[1] - st[0]) * a.G;
    if (rows > 0 && rows <= a.item_rows) return;
    // items are in the order of the blocks: the first one of block j
    const int32_t* it = a.items + (size_t)bh * a.max_items * 2;
    const int total = a.n_items[bh];
    int lo = 0, hi = total;
    while (lo < hi) {
        const int m = (lo + hi) / 2;
        if (it[2 * m] < j) lo = m + 1;
        else hi = m;
    }
    int end = lo;
    while (end < total && it[2 * end] == j) ++end;
    for (int i = threadIdx.x; i < 2 * kKeys * D / 4; i += 256) {
        const int which = i / (kKeys * D / 4), key = i % (kKeys * D / 4) / (D / 4), d = i % (D / 4) * 4, t = j * kKeys + key;
        if (t >= a.Nk) continue;
        f32x4 x{0.f, 0.f, 0.f, 0.f};
        for (int e = lo; e < end; ++e) x += *reinterpret_cast<const f32x4*>(a.slab + ((size_t)bh * a.max_items + e) * 2 * kKeys * D + (size_t)i * 4);
        T* dst = static_cast<T*>(which ? a.dv : a.dk);
        if (dst) tok_store4(dst + (((size_t)b * a.Nk + t) * a.KV + h) * D + d, x);
    }
}

// dQ: the n places of a query added
template <typename T, int D>
__global__ __launch_bounds__(256) void bs_dq_kernel(BsArgs a, long long rows) {
    constexpr int L = D / 4;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int sub = threadIdx.x % L;
    if (r >= rows) return;
    const unsigned hq = (unsigned)(r % a.H);
    const int32_t* bl = a.blocks + (r / a.H * a.KV + hq / (unsigned)a.G) * a.n;
    const float* part = static_cast<const float*>(a.part) + r * a.n * D + sub * 4;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < a.n; ++s)
        if (bl[s] >= 0 && bl[s] < a.NB) o += *reinterpret_cast<const f32x4*>(part + (long long)s * D);
    tok_store4(static_cast<T*>(a.dq) + r * D + sub * 4, o);
}

// ------------------------------------------------------------------------------------------------------------ host
constexpr int kMaxBlocks = 32768;            // LDS counters of the list kernels: 128 KB
constexpr int64_t kMaxRows = 0x7fffffff - 4 * kItemRows;      // rows of a block's list: loops step past the last one

int bs_check(const char* what, int32_t B, int32_t T, int32_t Nk, int32_t H, int32_t KV, int32_t D, int32_t n, int32_t dtype) {
    if (D != 16 && D != 32 && D != 64 && D != 128) return av2x::fail("%s: dim %d is not 16, 32, 64 or 128", what, D);
    if (dtype < 0 || dtype > 2) return av2x::fail("%s: dtype %d", what, dtype);
    if (B < 1 || T < 0 || Nk < 0 || H < 1 || KV < 1 || H % KV) return av2x::fail("%s: batch %d, queries %d, keys %d, heads %d over %d", what, B, T, Nk, H, KV);
    if (H / KV > 16 || H / KV * D > 1024) return av2x::fail("%s: %d heads of %d channels share keys (at most 16, 1024 channels)", what, H / KV, D);
    if (n < 1 || n > kMaxPick) return av2x::fail("%s: %d blocks a query (1 .. %d)", what, n, kMaxPick);
    if ((Nk + kKeys - 1) / kKeys > kMaxBlocks) return av2x::fail("%s: %d keys (at most %d)", what, Nk, kMaxBlocks * kKeys);
    if (T > (1 << 25) || (int64_t)T * n * (H / KV) > kMaxRows || B > 65535 / KV) return av2x::fail("%s: too many queries", what);
    return 0;
}

// rows are read in pieces of 16 bytes
int bs_rows(const char* what, const void* p, const int64_t* s, int dtype) {
    if (!p) return av2x::fail("%s: null tensor", what);
    const int64_t v = 16 / (int64_t)tok_size(dtype);
    if (!tok_aligned(p, 16) || s[0] % v || s[1] % v || s[2] % v) return av2x::fail("%s: tensors and strides must be aligned to 16 bytes", what);
    return 0;
}

int bs_runs(int64_t bh, int64_t entries) {
    int64_t r = 1024 / bh;
    const int64_t most = (entries + 255) / 256;
    if (r > most) r = most;
    return (int)(r < 1 ? 1 : r);
}

struct Lists { int32_t *hist, *start, *list, *items, *n_items; int runs, max_items, item_rows; size_t bytes; };
Lists bs_lists(void* base, int32_t B, int32_t T, int32_t Nk, int32_t H, int32_t KV, int32_t n) {
    Lists l{};
    const int64_t bh = (int64_t)B * KV, NB = (Nk + kKeys - 1) / kKeys, entries = (int64_t)T * n, rows = entries * (H / KV);
    l.runs = bs_runs(bh, entries);
    l.item_rows = (int)std::min<int64_t>(kItemRows, std::max<int64_t>(kItemLeast, bh * rows / 1024 / 128 * 128));
    l.max_items = (int)(rows / l.item_rows + NB + 1);
    int32_t* p = static_cast<int32_t*>(base);
    size_t at = 0;
    auto take = [&](int64_t count) { int32_t* r = p ? p + at : nullptr; at += (size_t)((count + 3) & ~3ll); return r; };
    l.list = take(bh * entries);
    l.start = take(bh * (NB + 1));
    l.items = take(bh * l.max_items * 2);
    l.n_items = take(bh);
    l.hist = take(bh * l.runs * NB);
    l.bytes = at * 4;
    return l;
}

template <typename F> int bs_go(int dtype, int dim, F&& f) {
    auto by_dim = [&](auto t) {
        switch (dim) {
            case 16: return f(t, std::integral_constant<int, 16>{});
            case 32: return f(t, std::integral_constant<int, 32>{});
            case 64: return f(t, std::integral_constant<int, 64>{});
            default: return f(t, std::integral_constant<int, 128>{});
        }
    };
    struct F32 { using type = float; };
    struct B16 { using type = __bf16; };
    struct H16 { using type = _Float16; };
    return dtype == kTokF32 ? by_dim(F32{}) : dtype == kTokBF16 ? by_dim(B16{}) : by_dim(H16{});
}

}  // namespace

extern "C" int av2x_block_bounds(const void* k, const uint8_t* mask, const int64_t* strides, int32_t batch, int32_t keys, int32_t kv_heads, int32_t dim, int32_t dtype,
                                 int32_t first_block, int32_t n_blocks, uint16_t* ints, float* scale, av2x_stream_t stream) {
    const char* what = "av2x_block_bounds";
    if (int rc = bs_check(what, batch, 0, keys, kv_heads, kv_heads, dim, 1, dtype)) return rc;
    const int NB = (keys + kKeys - 1) / kKeys;
    if (first_block < 0 || n_blocks < 0 || first_block > NB - n_blocks) return av2x::fail("%s: blocks %d .. %d of %d", what, first_block, first_block + n_blocks, NB);
    if (n_blocks == 0) return 0;
    if (!k || !ints || !scale) return av2x::fail("%s: null tensor", what);
    const size_t al = 4 * tok_size(dtype);
    if (!tok_aligned(k, al) || strides[0] % 4 || strides[1] % 4 || strides[2] % 4 || !tok_aligned(ints, 8)) return av2x::fail("%s: tensors and strides must be aligned to four elements", what);
    const long long total = (long long)batch * n_blocks * kv_heads;
    return bs_go(dtype, dim, [&](auto t, auto d) {
        using T = typename decltype(t)::type;
        bs_bounds_kernel<T, decltype(d)::value><<<(unsigned)((total + 3) / 4), 256, 0, av2x::as_stream(stream)>>>(
            static_cast<const T*>(k), mask, strides[0], strides[1], strides[2], keys, kv_heads, NB, first_block, n_blocks, reinterpret_cast<_Float16*>(ints), scale, total);
        return av2x::check_launch(what);
    });
}

namespace {

// Few queries leave the chip idle while a workgroup walks the scores of all blocks: the blocks are cut into ranges of whole chunks until there are
// about two workgroups a CU, and the ranges' choices joined (one query against 4400 blocks: 9 ranges of one chunk).  Measured (us, ranges / one walk):
// 8 heads of 32, 2200 blocks, n = 8: 1 query 13 / 20, 256: 18 / 23, 496 (the last before the rule): 25 / 24; n = 24: 35 / 84, 60 / 88, 62 / 88;
// 4 heads of 128: n = 8: 20 / 44, 27 / 57, 45 / 56
int select_parts(int64_t B, int64_t T, int64_t KV, int64_t NB) {
    const int64_t groups = (T + 15) / 16 * KV * B, chunks = (NB + kChunk - 1) / kChunk;
    if (chunks < 2 || groups >= 256) return 1;
    const int64_t want = (512 + groups - 1) / groups;
    return (int)(want < chunks ? want : chunks);
}

}  // namespace

extern "C" uint64_t av2x_select_blocks_workspace_bytes(int32_t batch, int32_t queries, int32_t keys, int32_t kv_heads, int32_t n) {
    if (batch < 1 || queries < 1 || keys < 0 || kv_heads < 1 || n < 1) return 0;
    const int p = select_parts(batch, queries, kv_heads, (keys + kKeys - 1) / kKeys);
    return p == 1 ? 0 : (uint64_t)batch * queries * kv_heads * p * n * sizeof(uint2);
}

extern "C" int av2x_select_blocks(const void* q, const int64_t* strides, const uint16_t* ints, const float* scale, int32_t batch, int32_t queries, int32_t keys,
                                  int32_t heads, int32_t kv_heads, int32_t dim, int32_t n, int32_t dtype, int32_t* blocks, void* workspace, av2x_stream_t stream) {
    const char* what = "av2x_select_blocks";
    if (int rc = bs_check(what, batch, queries, keys, heads, kv_heads, dim, n, dtype)) return rc;
    if (queries == 0) return 0;
    const int NB = (keys + kKeys - 1) / kKeys, parts = select_parts(batch, queries, kv_heads, NB);
    if (!q || !blocks || (NB && (!ints || !scale)) || (parts > 1 && !workspace)) return av2x::fail("%s: null tensor", what);
    if (!tok_aligned(ints, 16) || !tok_aligned(workspace, 8)) return av2x::fail("%s: the bounds must be aligned to 16 bytes", what);
    const int per = ((NB + parts - 1) / parts + kChunk - 1) / kChunk * kChunk, used = parts > 1 ? (NB + per - 1) / per : 1;
    hipStream_t st = av2x::as_stream(stream);
    return bs_go(dtype, dim, [&](auto t, auto d) {
        using T = typename decltype(t)::type;
        constexpr int D = decltype(d)::value;
        const _Float16* ip = reinterpret_cast<const _Float16*>(ints);
        auto go = [&](auto kernel, int nq, int parts_, int per_, int32_t* out, uint2* part) {
            kernel<<<dim3((unsigned)((queries + nq - 1) / nq) * parts_, kv_heads, batch), nq * 16, 0, st>>>(static_cast<const T*>(q), strides[0], strides[1], strides[2], ip, scale, queries,
                                                                                                      heads / kv_heads, kv_heads, NB, n, parts_, per_, out, part);
            return av2x::check_launch(what);
        };
        if (used == 1) return n <= 16 ? go(bs_select16_kernel<T, D, false>, 32, 1, NB, blocks, nullptr) : go(bs_select_kernel<T, D, false>, 16, 1, NB, blocks, nullptr);
        uint2* ws = static_cast<uint2*>(workspace);
        if (int rc = n <= 16 ? go(bs_select16_kernel<T, D, true>, 32, used, per, nullptr, ws) : go(bs_select_kernel<T, D, true>, 16, used, per, nullptr, ws)) return rc;
        bs_select_join_kernel<<<(unsigned)(batch * queries * kv_heads), 64, 0, st>>>(static_cast<const uint2*>(workspace), used, n, blocks);
        return av2x::check_launch(what);
    });
}

extern "C" uint64_t av2x_block_lists_bytes(int32_t batch, int32_t queries, int32_t keys, int32_t heads, int32_t kv_heads, int32_t n) {
    if (batch < 1 || queries < 0 || keys < 0 || kv_heads < 1 || heads < 1 || n < 1) return 0;
    return bs_lists(nullptr, batch, queries, keys, heads, kv_heads, n).bytes;
}

extern "C" int av2x_block_lists(const int32_t* blocks, int32_t batch, int32_t queries, int32_t keys, int32_t heads, int32_t kv_heads, int32_t n, void* lists,
                                av2x_stream_t stream) {
    const char* what = "av2x_block_lists";
    if (int rc = bs_check(what, batch, queries, keys, heads, kv_heads, 16, n, 0)) return rc;
    const int NB = (keys + kKeys - 1) / kKeys, bh = batch * kv_heads, G = heads / kv_heads;
    if (queries == 0 || NB == 0) return 0;
    if (!blocks || !lists || !tok_aligned(lists, 16)) return av2x::fail("%s: null or unaligned tensor", what);
    const Lists l = bs_lists(lists, batch, queries, keys, heads, kv_heads, n);
    const int64_t entries = (int64_t)queries * n;
    const int run_len = (int)(((entries + l.runs - 1) / l.runs + 63) / 64 * 64);
    int bits = 1;
    while (bits < 31 && NB > 1 << bits) ++bits;
    const size_t lds = (size_t)NB * 4;
    hipStream_t st = av2x::as_stream(stream);
    static av2x::LdsLimit lim0, lim1;
    if (lds > 65536) {                                   // one limit for all sizes: calls of other threads never lower it
        lim0.ensure((const void*)bs_count_kernel, kMaxBlocks * 4);
        lim1.ensure((const void*)bs_fill_kernel<1>, kMaxBlocks * 4);
    }
    bs_count_kernel<<<dim3(l.runs, bh), 256, lds, st>>>(blocks, queries, kv_heads, NB, n, l.runs, run_len, l.hist);
    if (int rc = av2x::check_launch(what)) return rc;
    bs_places_kernel<<<dim3((NB + 63) / 64, bh), 1024, 0, st>>>(l.hist, l.runs, NB, l.start);
    if (int rc = av2x::check_launch(what)) return rc;
    bs_scan_kernel<<<bh, 1024, 0, st>>>(NB, G, l.item_rows, l.max_items, l.start, l.items, l.n_items);
    if (int rc = av2x::check_launch(what)) return rc;
    if (4 * lds <= 65536) bs_fill_kernel<4><<<dim3(l.runs, bh), 256, 4 * lds, st>>>(blocks, queries, kv_heads, NB, n, l.runs, run_len, bits, l.hist, l.start, l.list);
    else bs_fill_kernel<1><<<dim3(l.runs, bh), 64, lds, st>>>(blocks, queries, kv_heads, NB, n, l.runs, run_len, bits, l.hist, l.start, l.list);
    return av2x::check_launch(what);
}

namespace {

size_t up16(size_t x) { return (x + 15) & ~(size_t)15; }

struct Work { size_t part, ld, slab, bytes; };       // byte offsets
Work bs_work(int64_t B, int64_t T, int64_t Nk, int64_t H, int64_t KV, int64_t D, int64_t n, bool backward) {
    Work w{};
    const size_t rows = (size_t)(B * T * H);
    w.part = 0;
    size_t at = up16(rows * n * (backward ? D * 4 : D * 4 + 8));
    if (backward) {
        w.ld = at;
        at += up16(rows * 8);
        w.slab = at;
        at += (size_t)bs_lists(nullptr, (int32_t)B, (int32_t)T, (int32_t)Nk, (int32_t)H, (int32_t)KV, (int32_t)n).max_items * B * KV * 2 * kKeys * D * 4;
    }
    w.bytes = at;
    return w;
}

BsArgs bs_args(const void* q, const void* k, const void* v, const uint8_t* mask, const int32_t* blocks, const void* lists, const int64_t* s, float scale, int32_t B,
               int32_t T, int32_t Nk, int32_t H, int32_t KV, int32_t n) {
    BsArgs a{};
    a.q = q; a.k = k; a.v = v; a.mask = mask; a.blocks = blocks;
    a.qb = s[0]; a.qt = s[1]; a.qh = s[2]; a.kb = s[3]; a.kt = s[4]; a.kh = s[5]; a.vb = s[6]; a.vt = s[7]; a.vh = s[8];
    a.B = B; a.T = T; a.Nk = Nk; a.H = H; a.KV = KV; a.G = H / KV; a.NB = (Nk + kKeys - 1) / kKeys; a.n = n;
    a.scale = scale;
    if (lists) {
        const Lists l = bs_lists(const_cast<void*>(lists), B, T, Nk, H, KV, n);
        a.list = l.list; a.start = l.start; a.items = l.items; a.n_items = l.n_items; a.max_items = l.max_items; a.item_rows = l.item_rows;
    }
    return a;
}

}  // namespace

extern "C" uint64_t av2x_block_sparse_workspace_bytes(int32_t batch, int32_t queries, int32_t keys, int32_t heads, int32_t kv_heads, int32_t dim, int32_t n, int32_t backward) {
    if (batch < 1 || queries < 0 || keys < 0 || kv_heads < 1 || heads < 1 || n < 1 || dim < 1) return 0;
    return bs_work(batch, queries, keys, heads, kv_heads, dim, n, backward != 0).bytes;
}

extern "C" int av2x_block_sparse_attention(const void* q, const void* k, const void* v, const int64_t* strides, const uint8_t* mask, const int32_t* blocks,
                                           const void* lists, int32_t batch, int32_t queries, int32_t keys, int32_t heads, int32_t kv_heads, int32_t dim, int32_t n,
                                           int32_t dtype, float scale, void* out, float* lse, void* rest, void* workspace, av2x_stream_t stream) {
    const char* what = "av2x_block_sparse_attention";
    if (int rc = bs_check(what, batch, queries, keys, heads, kv_heads, dim, n, dtype)) return rc;
    if (queries == 0) return 0;
    if (!out || !blocks || !workspace || !tok_aligned(out, 16) || !tok_aligned(workspace, 16) || !tok_aligned(lists, 16) || !tok_aligned(rest, 16)) return av2x::fail("%s: null or unaligned tensor", what);
    if (keys > 0) {
        if (int rc = bs_rows(what, q, strides, dtype)) return rc;
        if (int rc = bs_rows(what, k, strides + 3, dtype)) return rc;
        if (int rc = bs_rows(what, v, strides + 6, dtype)) return rc;
    }
    const long long mentions = (long long)batch * queries * kv_heads * n;
    if (!lists && mentions > 1 << 25) return av2x::fail("%s: so many queries need lists", what);
    BsArgs a = bs_args(q, k, v, mask, blocks, lists, strides, scale, batch, queries, keys, heads, kv_heads, n);
    const Work w = bs_work(batch, queries, keys, heads, kv_heads, dim, n, false);
    char* ws = static_cast<char*>(workspace);
    a.part = ws + w.part;
    a.out = out;
    a.lse = lse;
    a.rest = rest;
    hipStream_t st = av2x::as_stream(stream);
    return bs_go(dtype, dim, [&](auto t, auto d) {
        using T = typename decltype(t)::type;
        constexpr int D = decltype(d)::value;
        if (a.NB > 0) {
            const dim3 items(a.max_items, batch * kv_heads);
            if (lists) bs_forward_kernel<T, D><<<items, 256, 0, st>>>(a);
            else bs_few_kernel<T, D><<<(unsigned)mentions, 64, 0, st>>>(a);
            if (int rc = av2x::check_launch(what)) return rc;
        }
        const long long rows = (long long)batch * queries * heads;
        const unsigned by_row = (unsigned)((rows * (D / 4) + 255) / 256);
        bs_join_kernel<T, D><<<by_row, 256, 0, st>>>(a, rows);
        return av2x::check_launch(what);
    });
}

extern "C" int av2x_block_sparse_attention_backward(const void* q, const void* k, const void* v, const int64_t* strides, const uint8_t* mask, const int32_t* blocks,
                                                    const void* lists, const void* out, const void* rest, const float* lse, const void* dout, int32_t batch, int32_t queries, int32_t keys,
                                                    int32_t heads, int32_t kv_heads, int32_t dim, int32_t n, int32_t dtype, float scale, void* dq, void* dk, void* dv,
                                                    void* workspace, av2x_stream_t stream) {
    const char* what = "av2x_block_sparse_attention_backward";
    if (int rc = bs_check(what, batch, queries, keys, heads, kv_heads, dim, n, dtype)) return rc;
    if (queries == 0 || keys == 0) return av2x::fail("%s: no queries or no keys", what);
    const void* ptrs[] = {blocks, lists, out, lse, dout, workspace, dq};
    for (const void* p : ptrs)
        if (!p || !tok_aligned(p, 16)) return av2x::fail("%s: null or unaligned tensor", what);
    if (!tok_aligned(dk, 16) || !tok_aligned(dv, 16) || !tok_aligned(rest, 16)) return av2x::fail("%s: unaligned tensor", what);
    if (int rc = bs_rows(what, q, strides, dtype)) return rc;
    if (int rc = bs_rows(what, k, strides + 3, dtype)) return rc;
    if (int rc = bs_rows(what, v, strides + 6, dtype)) return rc;
    BsArgs a = bs_args(q, k, v, mask, blocks, lists, strides, scale, batch, queries, keys, heads, kv_heads, n);
    const Work w = bs_work(batch, queries, keys, heads, kv_heads, dim, n, true);
    char* ws = static_cast<char*>(workspace);
    f32x2* ld = reinterpret_cast<f32x2*>(ws + w.ld);
    a.part = ws + w.part;
    a.slab = reinterpret_cast<float*>(ws + w.slab);
    a.ld = ld;
    a.dout = dout;
    a.dq = dq; a.dk = dk; a.dv = dv;
    hipStream_t st = av2x::as_stream(stream);
    return bs_go(dtype, dim, [&](auto t, auto d) {
        using T = typename decltype(t)::type;
        constexpr int D = decltype(d)::value, DA = D <= 64 ? D : 64;      // heads of 128: what fits LDS and registers
        const long long rows = (long long)batch * queries * heads;
        const unsigned by_row = (unsigned)((rows * (D / 4) + 255) / 256);
        bs_delta_kernel<T, D><<<by_row, 256, 0, st>>>(static_cast<const T*>(out), static_cast<const T*>(rest), static_cast<const T*>(dout), lse, ld, rows);
        if (int rc = av2x::check_launch(what)) return rc;
        bs_backward_kernel<T, D, DA><<<dim3(a.max_items, batch * kv_heads, D / DA), 256, 0, st>>>(a);
        if (int rc = av2x::check_launch(what)) return rc;
        bs_dq_kernel<T, D><<<by_row, 256, 0, st>>>(a, rows);
        if (int rc = av2x::check_launch(what)) return rc;
        if (!dk && !dv) return 0;
        bs_dkv_kernel<T, D><<<dim3(a.NB, batch * kv_heads), 256, 0, st>>>(a);
        return av2x::check_launch(what);
    });
}
