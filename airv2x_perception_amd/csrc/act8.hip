// Saved activations in 8 bits and the backward passes that read them.
//
//   x8 = q s,  s = max|x| / 127 per row and group of 128 channels,  q = clamp(rint(x (127 / max(max|x|, 1e-30))), -127, 127)
//   (all three one correctly rounded fp32 operation each, so a stored byte does not depend on who computes it; a group that holds an
//   infinity or a NaN gets s = NaN: what was lost in the forward shows in the gradients)
//
//   act8_pack / act8_unpack          x -> (q, s), (q, s) -> x8                                                              HBM-bound
//   act8_layernorm                   y = (x - mean) rstd gamma + beta, (q, s) of x, (mean, rstd)   one pass over x          HBM-bound
//   act8_layernorm_backward          u = (x8 - mean) rstd, a = g gamma: dx = rstd (a - mean(a) - u mean(a u))               HBM-bound
//   act8_gelu / act8_gelu_backward   h = gelu(z) and (q, s) of z; dz = dh gelu'(z8)                                          HBM-bound
//   act8_wgrad                       dW = dY^T X over the rows, db = sum dY, X = x8 | u gamma + beta | gelu(x8)             matrix cores / HBM
//
// The weight gradient is where the bytes pay twice: an integer up to 127 is exact in bf16, so the scale moves to dY's side
// (dY s, split into three bf16 terms: exact to 2^-24) and a product costs three MFMAs where two fp32 operands cost six.
// Measured at 140800 rows of 256 channels: pack + GELU 58 us (330 MB, 5.7 TB/s), its backward 54 us; LayerNorm 71 us (4.7 TB/s), its backward 53 us (325 MB, part of it still
// in the caches); weight gradient of LayerNorm -> 768 outputs 270 us (166 GFLOP of bf16 products, 0.61 PFLOP/s), of GELU -> 256 183 us (111 GFLOP, 0.61 PFLOP/s):
// counters (norm / GELU): the matrix cores are busy in 37 / 33 % of the cycles, vector instructions -- the conversions between the products -- issue in 42 / 54 %, and LDS
// bank conflicts take 25 / 17 %: bound by the three taking turns at two waves a SIMD.
// LayerNorm's affine leaves the sum:  dW[o, i] = gamma_i (sum (dY s rstd)[r, o] q[r, i] - sum dY[r, o] mean_r rstd_r) + beta_i db_o.
#include <type_traits>

#include "token_common.hpp"

namespace {

constexpr int kGroup = 128;           // channels of one scale = columns of one weight-gradient tile
constexpr float kTiny = 1e-30f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// GELU from the normal tail:  Phi(-|z|) = exp(-z^2 / 2) t Q(t),  t = 1 / (1 + 0.3 |z|)  (the form of Abramowitz & Stegun 7.1.26; Q of degree 7 fitted here to
// 5e-8 of the tail).  With fp32 arithmetic a tail is off by at most 2^-21 + 1.5 z^2 2^-24 of itself: the exponent z^2 / 2 log2 e is rounded three times, and its error grows
// with it (measured: 4e-7 up to |z| = 2, 9e-7 to 4, 3e-6 to 8, 7e-6 to 12).  gelu(z) = z - z Phi(-z) or z Phi(z) then keeps its relative precision for negative z up to that,
// and the derivative shares the exponential.  16 instructions where erff and expf take about 90; the weight gradient evaluates it once per element and output tile.
__device__ __forceinline__ float normal_tail(float a, float& e) {      // a = |z|; e = exp(-z^2 / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.0f));
    float q = 0.037535473704338074f;
    q = fmaf(q, t, -0.16501864790916443f);
    q = fmaf(q, t, 0.21996943652629852f);
    q = fmaf(q, t, -0.06640082597732544f);
    q = fmaf(q, t, 0.13541917502880096f);
    q = fmaf(q, t, 0.09778428077697754f);
    q = fmaf(q, t, 0.12110564112663269f);
    q = fmaf(q, t, 0.11960549652576447f);
    e = __builtin_amdgcn_exp2f(-0.7213475204444817f * a * a);
    return q * t * e;
}
__device__ __forceinline__ float gelu8_f(float z) {
    float e;
    const float c = normal_tail(fabsf(z), e);
    return z < 0.f ? z * c : c == 0.f ? z : fmaf(-z, c, z);           // c == 0: infinity stays infinity
}
__device__ __forceinline__ float gelu8_df(float z) {
    float e;
    const float c = normal_tail(fabsf(z), e);
    return fmaf(z * 0.3989422804014327f, e, z < 0.f ? c : 1.0f - c);
}

// the 32 lanes of a group agree on its scale and quantise their four channels each
__device__ __forceinline__ unsigned pack4(f32x4 v, bool in, float* scale_out, int lane) {
    float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
    int bad = !(m < INFINITY) || v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;      // fmaxf skips a NaN
    if (!in) { m = 0.f; bad = 0; }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        m = fmaxf(m, __shfl_xor(m, o));
        bad |= __shfl_xor(bad, o);
    }
    const float r = 127.0f / fmaxf(m, kTiny);
    if (scale_out && (lane & 31) == 0) *scale_out = bad ? __builtin_nanf("") : m / 127.0f;
    auto q = [&](float x) { return (unsigned)(unsigned char)(signed char)(int)fminf(fmaxf(rintf(x * r), -127.f), 127.f); };
    return q(v.x) | q(v.y) << 8 | q(v.z) << 16 | q(v.w) << 24;
}

__device__ __forceinline__ f32x4 unpack4(unsigned w, float s) {
    return f32x4{(float)(signed char)(w & 0xff) * s, (float)(signed char)(w >> 8 & 0xff) * s, (float)(signed char)(w >> 16 & 0xff) * s,
                 (float)(signed char)(w >> 24) * s};
}

// One half wave per (row, group).  MODE 0: pack.  1: out = gelu(x) too.  2: unpack.  3: out = dy gelu'(x8).
template <int MODE>
__global__ __launch_bounds__(256) void act8_elementwise_kernel(const float* __restrict__ x, const float* __restrict__ dy, unsigned* __restrict__ q,
                                                               float* __restrict__ s, float* __restrict__ out, long long rows, int c) {
    const int groups = (c + kGroup - 1) / kGroup, lane = threadIdx.x & 63, l = lane & 31;
    const long long total = rows * groups, step = (long long)gridDim.x * 8;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += step) {      // a half wave leaves as one
        const long long row = i / groups;
        const int g = (int)(i - row * groups), ch = g * kGroup + l * 4;
        const bool in = ch < c;
        const size_t at = (size_t)row * c + ch;
        if constexpr (MODE <= 1) {
            f32x4 v{0.f, 0.f, 0.f, 0.f};
            if (in) v = *reinterpret_cast<const f32x4*>(x + at);
            const unsigned w = pack4(v, in, s + i, lane);
            if (in) {
                q[at / 4] = w;
                if constexpr (MODE == 1) *reinterpret_cast<f32x4*>(out + at) = f32x4{gelu8_f(v.x), gelu8_f(v.y), gelu8_f(v.z), gelu8_f(v.w)};
            }
        } else if (in) {
            f32x4 v = unpack4(q[at / 4], s[i]);
            if constexpr (MODE == 3) {
                const f32x4 d = *reinterpret_cast<const f32x4*>(dy + at);
                v = f32x4{d.x * gelu8_df(v.x), d.y * gelu8_df(v.y), d.z * gelu8_df(v.z), d.w * gelu8_df(v.w)};
            }
            *reinterpret_cast<f32x4*>(out + at) = v;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ LayerNorm
// one wave per row, 256 CK channels at most; channel k * 256 + lane * 4: the two half waves of a step are two groups
template <int CK>
__global__ __launch_bounds__(256) void act8_layernorm_kernel(const float* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             float* __restrict__ y, unsigned* __restrict__ q, float* __restrict__ s,
                                                             f32x2* __restrict__ stats, long long rows, int c, float eps) {
    const int lane = threadIdx.x & 63, groups = (c + kGroup - 1) / kGroup;
    for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long long)gridDim.x * 4) {
        f32x4 v[CK];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            const int ch = k * 256 + lane * 4;
            v[k] = ch < c ? *reinterpret_cast<const f32x4*>(x + (size_t)row * c + ch) : f32x4{0.f, 0.f, 0.f, 0.f};
            sum += (v[k].x + v[k].y) + (v[k].z + v[k].w);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
        const float mean = sum / (float)c;
        float sq = 0.f;
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            if (k * 256 + lane * 4 < c) {
                const f32x4 d = v[k] - mean;
                sq += (d.x * d.x + d.y * d.y) + (d.z * d.z + d.w * d.w);
            }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sq += __shfl_xor(sq, o);
        const float rstd = 1.0f / sqrtf(sq / (float)c + eps);
        if (lane == 0) stats[row] = f32x2{mean, rstd};
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            const int ch = k * 256 + lane * 4, g = ch / kGroup;
            const bool in = ch < c;
            const unsigned w = pack4(v[k], in, in ? s + row * groups + g : nullptr, lane);
            if (in) {
                const size_t at = (size_t)row * c + ch;
                q[at / 4] = w;
                *reinterpret_cast<f32x4*>(y + at) = (v[k] - mean) * rstd * *reinterpret_cast<const f32x4*>(gamma + ch) + *reinterpret_cast<const f32x4*>(beta + ch);
            }
        }
    }
}

// dx alone: the gradients of gamma and beta come out of the weight gradient (act8_affine_kernel)
template <int CK>
__global__ __launch_bounds__(256) void act8_layernorm_backward_kernel(const unsigned* __restrict__ q, const float* __restrict__ s,
                                                                      const f32x2* __restrict__ stats, const float* __restrict__ gamma,
                                                                      const float* dy, float* dx, long long rows, int c) {      // dx may be dy
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = (c + kGroup - 1) / kGroup;
    f32x4 gm[CK];
#pragma unroll
    for (int k = 0; k < CK; ++k) {
        const int ch = k * 256 + lane * 4;
        gm[k] = ch < c ? *reinterpret_cast<const f32x4*>(gamma + ch) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (long long row = (long long)blockIdx.x * 4 + wave; row < rows; row += (long long)gridDim.x * 4) {
        const f32x2 st = stats[row];
        f32x4 u[CK], d[CK];
        float sa = 0.f, sb = 0.f;
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            const int ch = k * 256 + lane * 4;
            u[k] = d[k] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (ch < c) {
                const size_t at = (size_t)row * c + ch;
                u[k] = (unpack4(q[at / 4], s[row * groups + ch / kGroup]) - st.x) * st.y;
                d[k] = *reinterpret_cast<const f32x4*>(dy + at) * gm[k];
            }
            sa += (d[k].x + d[k].y) + (d[k].z + d[k].w);
            sb += (d[k].x * u[k].x + d[k].y * u[k].y) + (d[k].z * u[k].z + d[k].w * u[k].w);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) { sa += __shfl_xor(sa, o); sb += __shfl_xor(sb, o); }
        const float ma = sa / (float)c, mb = sb / (float)c;
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            const int ch = k * 256 + lane * 4;
            if (ch < c) *reinterpret_cast<f32x4*>(dx + (size_t)row * c + ch) = (d[k] - ma - u[k] * mb) * st.y;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ weight gradient
// Tile 128 outputs x 128 inputs (one scale group) x 32 rows, four waves of 64 x 64, two workgroups a CU; a workgroup walks its share of the rows and writes a slab;
// act8_wgrad_reduce_kernel adds the slabs in order.  The pieces of dY and q are transposed on the way to LDS: a thread loads four rows of four columns and
// writes, per column, its rows as half a fragment of an MFMA operand.  dY, q and the rows' scales of the next step are on their way during the products.
// The workgroups of one share of the rows have neighbouring numbers on one XCD: its L2 serves dY to all tiles of inputs and q to all tiles of outputs.
enum { kPlain = 0, kNorm = 1, kGelu = 2 };
// Element offset of eight rows of a column, 32 rows a column.  Pitch 80 bytes: sixteen neighbouring columns (readers) start in sixteen different 16-byte slots of the
// banks; every fourth column (writers) meets only four, so the fragment within a column turns with col / 16.
constexpr int kPitch = 40;
__device__ __forceinline__ int swz(int col, int chunk) { return col * kPitch + ((chunk ^ (col >> 4)) & 3) * 8; }

template <int N, typename V> __device__ __forceinline__ void split3(const float (&v)[N], V& hi, V& mid, V& lo) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        f32x2 a{v[i], v[i + 1]};
        const bf16x2 h = __builtin_convertvector(a, bf16x2);
        const f32x2 hf = __builtin_convertvector(h, f32x2);
        a.x -= hf.x; a.y -= hf.y;
        const bf16x2 m = __builtin_convertvector(a, bf16x2);
        const f32x2 mf = __builtin_convertvector(m, f32x2);
        a.x -= mf.x; a.y -= mf.y;
        const bf16x2 l = __builtin_convertvector(a, bf16x2);
        hi[i] = h[0]; hi[i + 1] = h[1];
        mid[i] = m[0]; mid[i + 1] = m[1];
        lo[i] = l[0]; lo[i + 1] = l[1];
    }
}

template <int KIND>
__global__ __launch_bounds__(256, 2) void act8_wgrad_kernel(const float* __restrict__ dy, const unsigned* __restrict__ q, const float* __restrict__ s,
                                                         const f32x2* __restrict__ stats, float* __restrict__ slabs, float* __restrict__ extra,
                                                         long long rows, int co, int ci, int tiles_o, int tiles_i, long long rows_per, int splits) {
    constexpr int XP = KIND == kGelu ? 3 : 1;                        // bf16 terms of X
    constexpr int R = 32, RT = R / 8;                                // rows of a step, of a thread
    constexpr int PLANE = 128 * kPitch;
    // two buffers where two workgroups of them just fill the 160 KB of a CU: one barrier a step, and a wave writes its part of the next step without waiting
    constexpr bool TWO = KIND != kGelu;
    constexpr int BUF = (3 + XP) * PLANE;
    typedef __bf16 bfv __attribute__((ext_vector_type(RT)));
    extern __shared__ __align__(16) char smem[];
    __bf16* la = reinterpret_cast<__bf16*>(smem);                    // [buffer][3][128][kPitch]
    __bf16* lb = la + 3 * PLANE;                                     // [buffer][XP][128][kPitch]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // workgroups go round the eight XCDs: number x of XCD c takes tile x % tiles of share 8 (x / tiles) + c
    const int tiles = tiles_o * tiles_i, xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
    const int tile = local % tiles, split = local / tiles * 8 + xcd;
    if (split >= splits) return;
    const int o0 = tile / tiles_i * 128, g = tile % tiles_i, i0 = g * 128, groups = tiles_i;
    const long long r0 = split * rows_per, r1 = min(rows, r0 + rows_per);
    const int cg = tid & 31, rc = tid >> 5;                          // four columns, RT rows
    const int oc = o0 + cg * 4, ic = i0 + cg * 4;
    const bool oin = oc < co;
    const int wo = (wave >> 1) * 64, wi = (wave & 1) * 64;
    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
    f32x4 sum{0.f, 0.f, 0.f, 0.f}, sumu{0.f, 0.f, 0.f, 0.f};
    struct Raw { f32x4 d[RT]; unsigned q[RT]; float s[RT]; f32x2 st[RT]; };
    // columns behind the last are read from the last ones: their results are not stored
    const float* dyp = dy + (size_t)(r0 + rc * RT) * co + min(oc, co - 4);
    const unsigned* qp = q + ((size_t)(r0 + rc * RT) * ci + min(ic, ci - 4)) / 4;
    const float* sp = s + (size_t)(r0 + rc * RT) * groups + g;
    const f32x2* tp = stats + (r0 + rc * RT);
    const int ciq = ci / 4;
    long long rf = r0;                                               // the step that is fetched next
    auto fetch = [&](Raw& w) {
        if (rf + R <= r1) {
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                w.d[j] = *reinterpret_cast<const f32x4*>(dyp + (size_t)j * co);
                w.q[j] = qp[(size_t)j * ciq];
                w.s[j] = sp[(size_t)j * groups];
                if constexpr (KIND == kNorm) w.st[j] = tp[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const bool in = rf + rc * RT + j < r1;
                w.d[j] = in ? *reinterpret_cast<const f32x4*>(dyp + (size_t)j * co) : f32x4{0.f, 0.f, 0.f, 0.f};
                w.q[j] = in ? qp[(size_t)j * ciq] : 0u;
                w.s[j] = in ? sp[(size_t)j * groups] : 0.f;
                if constexpr (KIND == kNorm) w.st[j] = in ? tp[j] : f32x2{0.f, 0.f};
            }
        }
        rf += R;
        dyp += (size_t)R * co;
        qp += (size_t)R * ciq;
        sp += (size_t)R * groups;
        tp += R;
    };
    bfv ta[4][3], tb[4][XP];                                         // one step's terms, per column
    auto convert = [&](const Raw& w, int e) {                        // column e of the four
        float v[RT], x[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            v[j] = KIND == kGelu ? w.d[j][e] : KIND == kNorm ? w.d[j][e] * (w.s[j] * w.st[j].y) : w.d[j][e] * w.s[j];
            x[j] = (float)(signed char)(w.q[j] >> (8 * e) & 0xff);
            if constexpr (KIND == kNorm) sumu[e] += w.d[j][e] * (w.st[j].x * w.st[j].y);
        }
        sum[e] += (w.d[0][e] + w.d[1][e]) + (w.d[2][e] + w.d[3][e]);
        split3<RT>(v, ta[e][0], ta[e][1], ta[e][2]);
        if constexpr (KIND == kGelu) {
#pragma unroll
            for (int j = 0; j < RT; ++j) x[j] = gelu8_f(x[j] * w.s[j]);
            split3<RT>(x, tb[e][0], tb[e][1], tb[e][2]);
        } else {
#pragma unroll
            for (int j = 0; j < RT; j += 2) {
                const bf16x2 h = __builtin_convertvector((f32x2{x[j], x[j + 1]}), bf16x2);     // |x| <= 127: exact
                tb[e][0][j] = h[0]; tb[e][0][j + 1] = h[1];
            }
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = buf * BUF + swz(cg * 4 + e, rc * RT / 8) + rc * RT % 8;
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<bfv*>(la + p * PLANE + at) = ta[e][p];
#pragma unroll
            for (int p = 0; p < XP; ++p) *reinterpret_cast<bfv*>(lb + p * PLANE + at) = tb[e][p];
        }
    };
    // one step: the one after next is fetched, the next one is converted between the products and goes to LDS
    auto step = [&](Raw& next, Raw& later, int buf) {
        fetch(later);
#pragma unroll
        for (int ks = 0; ks < R / 16; ++ks) {
            const int chunk = ks * 2 + (lane >> 5);
            bf16x8 A[2][3], B[2][XP];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int p = 0; p < 3; ++p) A[m][p] = *reinterpret_cast<const bf16x8*>(la + buf * BUF + p * PLANE + swz(wo + m * 32 + (lane & 31), chunk));
#pragma unroll
                for (int p = 0; p < XP; ++p) B[m][p] = *reinterpret_cast<const bf16x8*>(lb + buf * BUF + p * PLANE + swz(wi + m * 32 + (lane & 31), chunk));
            }
            // terms from the smallest products to the largest; the four tiles of a term follow each other, so that no product waits for the one before
            auto term = [&](int pa, int pb) {
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int b = 0; b < 2; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[a][pa], B[b][pb], acc[a][b], 0, 0, 0);
            };
            if constexpr (KIND == kGelu) {
                term(2, 0);
                term(0, 2);
                term(1, 1);
                convert(next, ks * 2);
                term(1, 0);
                term(0, 1);
            } else {
                term(2, 0);
                convert(next, ks * 2);
                term(1, 0);
            }
            convert(next, ks * 2 + 1);
            term(0, 0);
        }
        if constexpr (!TWO) __syncthreads();
        put(TWO ? buf ^ 1 : 0);
        __syncthreads();
    };
    if (r0 < r1) {
        Raw u, v;
        fetch(u);
#pragma unroll
        for (int e = 0; e < 4; ++e) convert(u, e);
        fetch(u);
        put(0);
        __syncthreads();
        const long long n = (r1 - r0 + R - 1) / R;                   // (two more are fetched and converted: zeros)
        for (long long i = 0; i < n; i += 2) {
            step(u, v, 0);
            if (i + 1 < n) step(v, u, TWO ? 1 : 0);
        }
    }
    __syncthreads();
    float* slab = slabs + (size_t)split * co * ci;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int o = o0 + wo + a * 32 + 8 * (e / 4) + 4 * (lane >> 5) + (e & 3), i = i0 + wi + b * 32 + (lane & 31);
                if (o < co && i < ci) slab[(size_t)o * ci + i] = acc[a][b][e];
            }
    if (g == 0) {                                                    // sums over the rows: once per output tile
        f32x4* red = reinterpret_cast<f32x4*>(smem);                 // [2][8][32]
        red[rc * 32 + cg] = sum;
        red[256 + rc * 32 + cg] = sumu;
        __syncthreads();
        if (tid < 64) {
            const int which = tid >> 5;
            f32x4 t = red[which * 256 + cg];
            for (int j = 1; j < 8; ++j) t += red[which * 256 + j * 32 + cg];
            if (oin) *reinterpret_cast<f32x4*>(extra + ((size_t)split * 2 + which) * co + oc) = t;
        }
    }
}

// dW of one output row and up to 256 inputs: four waves take every fourth slab each.  kNorm: the sum before LayerNorm's affine, sum dY u, is kept in `pre`
template <int KIND>
__global__ __launch_bounds__(256) void act8_wgrad_reduce_kernel(const float* __restrict__ slabs, const float* __restrict__ extra, int splits, int co, int ci,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta, float* __restrict__ dw,
                                                                float* __restrict__ db, float* __restrict__ pre) {
    __shared__ f32x4 red[4][64];
    __shared__ float rs[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, o = blockIdx.y, i = blockIdx.x * 256 + lane * 4;
    f32x4 t{0.f, 0.f, 0.f, 0.f};
    if (i < ci) {
#pragma unroll 4
        for (int sp = wave; sp < splits; sp += 4) t += *reinterpret_cast<const f32x4*>(slabs + ((size_t)sp * co + o) * ci + i);
    }
    red[wave][lane] = t;
    float e0 = 0.f, e1 = 0.f;
    for (int sp = threadIdx.x; sp < splits; sp += 256) {
        e0 += extra[((size_t)sp * 2) * co + o];
        e1 += extra[((size_t)sp * 2 + 1) * co + o];
    }
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) { e0 += __shfl_xor(e0, k); e1 += __shfl_xor(e1, k); }
    if (lane == 0) { rs[0][wave] = e0; rs[1][wave] = e1; }
    __syncthreads();
    if (wave == 0) {
        const float d = (rs[0][0] + rs[0][1]) + (rs[0][2] + rs[0][3]), u = (rs[1][0] + rs[1][1]) + (rs[1][2] + rs[1][3]);
        if (i < ci) {
            t = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
            if constexpr (KIND == kNorm) {
                t -= u;
                if (pre) *reinterpret_cast<f32x4*>(pre + (size_t)o * ci + i) = t;
                t = t * *reinterpret_cast<const f32x4*>(gamma + i) + *reinterpret_cast<const f32x4*>(beta + i) * d;
            }
            if (dw) *reinterpret_cast<f32x4*>(dw + (size_t)o * ci + i) = t;
        }
        if (blockIdx.x == 0 && lane == 0 && db) db[o] = d;
    }
}

// The affine's gradients without another pass over the rows:  dgamma_i = sum_r (dY W)[r, i] u[r, i] = sum_o W[o, i] (sum_r dY[r, o] u[r, i]),
// dbeta_i = sum_o W[o, i] db_o.  Also the more exact way: dY W itself is rounded row by row.  32 channels x 32 rows of outputs a workgroup.
__global__ __launch_bounds__(1024) void act8_affine_kernel(const float* __restrict__ w, const float* __restrict__ pre, const float* __restrict__ db, int co, int ci,
                                                           float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[2][32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, i = blockIdx.x * 32 + c;
    float g = 0.f, b = 0.f;
    if (i < ci) {
#pragma unroll 4
        for (int o = r; o < co; o += 32) {
            const float x = w[(size_t)o * ci + i];
            g += x * pre[(size_t)o * ci + i];
            b += x * db[o];
        }
    }
    red[0][r][c] = g;
    red[1][r][c] = b;
    __syncthreads();
    if (r < 2 && i < ci) {
        float t = 0.f;
        for (int k = 0; k < 32; ++k) t += red[r][k][c];
        float* out = r ? dbeta : dgamma;
        if (out) out[i] = t;
    }
}

// ------------------------------------------------------------------------------------------------------------ products for few rows
// Y (rows x n) = A (rows x k) B + bias + residual, all fp32, six products of three bf16 terms each (exact to 2^-24 as the framework's large GEMM), B read as the
// parameter lies: B = W^T of W (n, k) (forward) or W of W (k, n) (data gradient).  For few rows: the framework's GEMM wants W packed and split first, four
// launches and their host time where a step has new weights; tiles of 64 x 64 fill the chip sooner (2200 x 256 x 256: 9 us against 19
// with packing).  A tile's products are few: bound by the loads' latency and the split of both operands.
// TRANS: B is (k, n): a thread transposes two rows of four columns on the way to LDS.
constexpr int kSmallK = 32;
template <bool TRANS>
__global__ __launch_bounds__(256) void act8_gemm_kernel(const float* __restrict__ a, const float* __restrict__ w, const float* __restrict__ bias,
                                                        const float* __restrict__ residual, float* __restrict__ y, int rows, int n, int k) {
    constexpr int P = kSmallK + 8;                                   // row pitch: sixteen lanes meet all banks
    __shared__ __align__(16) __bf16 la[2][3][64 * P], lb[2][3][64 * P];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int r0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
    const int row = tid >> 2, kc = (tid & 3) * 8;                    // 64 rows x 4 pieces of eight k
    const int tk = (tid >> 4) * 2, tn = (tid & 15) * 4;              // TRANS: two k x four n
    const int ra = min(r0 + row, rows - 1), rb = min(n0 + row, n - 1);
    f32x4 pa[2], pb[2];
    auto fetch = [&](int k0) {
        const float* p = a + (size_t)ra * k + k0 + kc;
        pa[0] = *reinterpret_cast<const f32x4*>(p);
        pa[1] = *reinterpret_cast<const f32x4*>(p + 4);
        if constexpr (TRANS) {
            const float* p2 = w + (size_t)(k0 + tk) * n + min(n0 + tn, n - 4);
            pb[0] = *reinterpret_cast<const f32x4*>(p2);
            pb[1] = *reinterpret_cast<const f32x4*>(p2 + n);
        } else {
            const float* p2 = w + (size_t)rb * k + k0 + kc;
            pb[0] = *reinterpret_cast<const f32x4*>(p2);
            pb[1] = *reinterpret_cast<const f32x4*>(p2 + 4);
        }
    };
    auto stage = [&](int buf) {
        float v[8];
        bf16x8 t[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = pa[e >> 2][e & 3];
        split3<8>(v, t[0], t[1], t[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(&la[buf][p][row * P + kc]) = t[p];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = TRANS ? pb[e & 1][e >> 1] : pb[e >> 2][e & 3];
        split3<8>(v, t[0], t[1], t[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            if constexpr (TRANS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) *reinterpret_cast<bf16x2*>(&lb[buf][p][(tn + e) * P + tk]) = bf16x2{t[p][2 * e], t[p][2 * e + 1]};
            } else {
                *reinterpret_cast<bf16x8*>(&lb[buf][p][row * P + kc]) = t[p];
            }
        }
    };
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    const int m = (wave >> 1) * 32 + (lane & 31), c = (wave & 1) * 32 + (lane & 31);
    fetch(0);
    int buf = 0;
    for (int k0 = 0; k0 < k; k0 += kSmallK, buf ^= 1) {
        stage(buf);
        __syncthreads();                                             // the other buffer's readers are past it: one barrier a step
        if (k0 + kSmallK < k) fetch(k0 + kSmallK);
#pragma unroll
        for (int s = 0; s < kSmallK / 16; ++s) {
            bf16x8 A[3], B[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                A[p] = *reinterpret_cast<const bf16x8*>(&la[buf][p][m * P + s * 16 + half * 8]);
                B[p] = *reinterpret_cast<const bf16x8*>(&lb[buf][p][c * P + s * 16 + half * 8]);
            }
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[2], B[0], acc, 0, 0, 0);       // smallest first
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], acc, 0, 0, 0);
        }
    }
    const int col = n0 + c;
    if (col >= n) return;
    const float bv = bias ? bias[col] : 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int r = r0 + (wave >> 1) * 32 + 8 * (e / 4) + 4 * half + (e & 3);
        if (r >= rows) continue;
        float v = acc[e] + bv;
        if (residual) v += residual[(size_t)r * n + col];
        y[(size_t)r * n + col] = v;
    }
}

int act8_check(const char* what, const void* const* ptrs, int n, int64_t rows, int32_t c, int32_t most) {
    if (rows < 0 || rows > (1ll << 40)) return av2x::fail("%s: rows %lld", what, (long long)rows);
    if (c < 4 || c % 4 || c > most) return av2x::fail("%s: %d channels (a multiple of 4, at most %d)", what, c, most);
    for (int i = 0; i < n; ++i) {
        if (!ptrs[i]) return av2x::fail("%s: null tensor", what);
        if (!tok_aligned(ptrs[i], 16)) return av2x::fail("%s: tensors must be aligned to 16 bytes", what);
    }
    return 0;
}

unsigned act8_grid(int64_t half_waves) {
    const int64_t g = (half_waves + 7) / 8;
    return (unsigned)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

constexpr int kMaxC = 1 << 20;

struct WgradPlan { int tiles_o, tiles_i, splits; int64_t rows_per; };
WgradPlan wgrad_plan(int64_t rows, int co, int ci) {
    constexpr int kRows = 64;
    WgradPlan p{(co + 127) / 128, (ci + 127) / 128, 1, kRows};
    // two workgroups a CU; at least one step of rows each; whole rounds of the XCDs.  (us at 256 / 512 / 1024 shares x tiles: 140800 rows 256 -> 768: 404 / 219 / 229,
    // 35200 rows: 95 / 64 / 72, 8800 rows 256 -> 256: 23 / 25 / 31)
    int64_t want = 512 / ((int64_t)p.tiles_o * p.tiles_i);
    if (want > 8) want = want / 8 * 8;
    const int64_t steps = (rows + kRows - 1) / kRows;
    if (want > steps) want = steps;
    if (want < 1) want = 1;
    p.rows_per = (steps + want - 1) / want * kRows;
    if (p.rows_per < kRows) p.rows_per = kRows;
    p.splits = (int)((rows + p.rows_per - 1) / p.rows_per);
    if (p.splits < 1) p.splits = 1;
    return p;
}

}  // namespace

extern "C" int av2x_act8_pack(const float* x, int8_t* q, float* scale, int64_t rows, int32_t c, av2x_stream_t stream) {
    const void* p[] = {x, q, scale};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_pack", p, 3, rows, c, kMaxC)) return rc;
    act8_elementwise_kernel<0><<<act8_grid(rows * ((c + 127) / 128)), 256, 0, av2x::as_stream(stream)>>>(x, nullptr, (unsigned*)q, scale, nullptr, rows, c);
    return av2x::check_launch("av2x_act8_pack");
}

extern "C" int av2x_act8_unpack(const int8_t* q, const float* scale, float* out, int64_t rows, int32_t c, av2x_stream_t stream) {
    const void* p[] = {q, scale, out};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_unpack", p, 3, rows, c, kMaxC)) return rc;
    act8_elementwise_kernel<2><<<act8_grid(rows * ((c + 127) / 128)), 256, 0, av2x::as_stream(stream)>>>(nullptr, nullptr, (unsigned*)q, (float*)scale, out, rows, c);
    return av2x::check_launch("av2x_act8_unpack");
}

extern "C" int av2x_act8_gelu(const float* z, float* h, int8_t* q, float* scale, int64_t rows, int32_t c, av2x_stream_t stream) {
    const void* p[] = {z, h, q, scale};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_gelu", p, 4, rows, c, kMaxC)) return rc;
    act8_elementwise_kernel<1><<<act8_grid(rows * ((c + 127) / 128)), 256, 0, av2x::as_stream(stream)>>>(z, nullptr, (unsigned*)q, scale, h, rows, c);
    return av2x::check_launch("av2x_act8_gelu");
}

extern "C" int av2x_act8_gelu_backward(const int8_t* q, const float* scale, const float* dh, float* dz, int64_t rows, int32_t c, av2x_stream_t stream) {
    const void* p[] = {q, scale, dh, dz};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_gelu_backward", p, 4, rows, c, kMaxC)) return rc;
    act8_elementwise_kernel<3><<<act8_grid(rows * ((c + 127) / 128)), 256, 0, av2x::as_stream(stream)>>>(nullptr, dh, (unsigned*)q, (float*)scale, dz, rows, c);
    return av2x::check_launch("av2x_act8_gelu_backward");
}

extern "C" int av2x_act8_layernorm(const float* x, const float* gamma, const float* beta, float* y, int8_t* q, float* scale, float* stats, int64_t rows,
                                   int32_t c, float eps, av2x_stream_t stream) {
    const void* p[] = {x, gamma, beta, y, q, scale, stats};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_layernorm", p, 7, rows, c, 1024)) return rc;
    const unsigned grid = (unsigned)((rows + 3) / 4 < 8192 ? (rows + 3) / 4 : 8192);
    auto go = [&](auto ck) {
        act8_layernorm_kernel<decltype(ck)::value><<<grid, 256, 0, av2x::as_stream(stream)>>>(x, gamma, beta, y, (unsigned*)q, scale, (f32x2*)stats, rows, c, eps);
    };
    if (c <= 256) go(std::integral_constant<int, 1>{});
    else if (c <= 512) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    return av2x::check_launch("av2x_act8_layernorm");
}

extern "C" int av2x_act8_layernorm_backward(const int8_t* q, const float* scale, const float* stats, const float* gamma, const float* dy, float* dx, int64_t rows,
                                            int32_t c, av2x_stream_t stream) {
    const void* p[] = {gamma, q, scale, stats, dy, dx};
    if (rows == 0) return 0;
    if (int rc = act8_check("av2x_act8_layernorm_backward", p, 6, rows, c, 1024)) return rc;
    const unsigned grid = (unsigned)((rows + 3) / 4 < 8192 ? (rows + 3) / 4 : 8192);
    auto go = [&](auto ck) {
        act8_layernorm_backward_kernel<decltype(ck)::value><<<grid, 256, 0, av2x::as_stream(stream)>>>((const unsigned*)q, scale, (const f32x2*)stats, gamma, dy, dx, rows, c);
    };
    if (c <= 256) go(std::integral_constant<int, 1>{});
    else if (c <= 512) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    return av2x::check_launch("av2x_act8_layernorm_backward");
}

extern "C" uint64_t av2x_act8_wgrad_workspace_bytes(int64_t rows, int32_t cout, int32_t cin) {
    if (rows < 0 || cout < 1 || cin < 1) return 0;
    const WgradPlan p = wgrad_plan(rows, cout, cin);
    return ((uint64_t)(p.splits + 1) * cout * cin + (2ull * p.splits + 1) * cout) * 4;
}

extern "C" int av2x_act8_wgrad(const float* dy, const int8_t* q, const float* scale, const float* stats, const float* gamma, const float* beta, const float* weight,
                               int32_t kind, int64_t rows, int32_t cout, int32_t cin, float* dw, float* db, float* dgamma, float* dbeta, void* workspace,
                               av2x_stream_t stream) {
    const char* what = "av2x_act8_wgrad";
    const void* p[] = {workspace, dy, q, scale};
    if (kind < 0 || kind > 2) return av2x::fail("%s: kind %d", what, kind);
    if (int rc = act8_check(what, p, rows ? 4 : 1, rows, cin, 65536)) return rc;
    if (cout < 4 || cout % 4 || cout > 65532) return av2x::fail("%s: %d outputs (a multiple of 4, at most 65532)", what, cout);
    if (kind == kNorm && (!gamma || !beta || (rows && !stats))) return av2x::fail("%s: LayerNorm's statistics and parameters are needed", what);
    if ((dgamma || dbeta) && (kind != kNorm || !weight)) return av2x::fail("%s: the affine's gradients need LayerNorm (kind 1) and the weight", what);
    if (!tok_aligned(gamma, 16) || !tok_aligned(beta, 16) || !tok_aligned(dw, 16) || !tok_aligned(stats, 8)) return av2x::fail("%s: tensors must be aligned to 16 bytes", what);
    const WgradPlan pl = wgrad_plan(rows, cout, cin);
    float* slabs = static_cast<float*>(workspace);
    float* extra = slabs + (size_t)pl.splits * cout * cin;
    float* pre = extra + (size_t)2 * pl.splits * cout;
    float* dbw = db ? db : pre + (size_t)cout * cin;
    const int64_t grid = (int64_t)pl.tiles_o * pl.tiles_i * ((pl.splits + 7) / 8 * 8);
    if (grid > 0x7fffffff) return av2x::fail("%s: too large", what);
    const bool affine = dgamma || dbeta;
    hipStream_t st = av2x::as_stream(stream);
    auto go = [&](auto kd) {
        constexpr int K = decltype(kd)::value;
        constexpr size_t lds = (size_t)(K == kGelu ? 6 : 2 * 4) * 128 * kPitch * 2;
        static av2x::LdsLimit lim;
        lim.ensure((const void*)act8_wgrad_kernel<K>, lds);
        act8_wgrad_kernel<K><<<(unsigned)grid, 256, lds, st>>>(dy, (const unsigned*)q, scale, (const f32x2*)stats, slabs, extra, rows, cout, cin, pl.tiles_o, pl.tiles_i,
                                                             pl.rows_per, pl.splits);
        if (int rc = av2x::check_launch(what)) return rc;
        act8_wgrad_reduce_kernel<K><<<dim3((cin + 255) / 256, cout), 256, 0, st>>>(slabs, extra, pl.splits, cout, cin, gamma, beta, dw, affine ? dbw : db, affine ? pre : nullptr);
        if (int rc = av2x::check_launch("av2x_act8_wgrad: sums")) return rc;
        if (!affine) return 0;
        act8_affine_kernel<<<(cin + 31) / 32, 1024, 0, st>>>(weight, pre, dbw, cout, cin, dgamma, dbeta);
        return av2x::check_launch("av2x_act8_wgrad: affine");
    };
    if (kind == kPlain) return go(std::integral_constant<int, kPlain>{});
    if (kind == kNorm) return go(std::integral_constant<int, kNorm>{});
    return go(std::integral_constant<int, kGelu>{});
}

extern "C" int av2x_act8_gemm(const float* a, const float* w, const float* bias, const float* residual, float* y, int64_t rows, int32_t n, int32_t k, int32_t w_is_kn,
                              av2x_stream_t stream) {
    const char* what = "av2x_act8_gemm";
    const void* p[] = {a, w, y};
    if (rows == 0) return 0;
    if (int rc = act8_check(what, p, 3, rows, k, 65536)) return rc;
    if (k % 32 || n < 4 || n % 4 || n > 65536 * 32 || rows > (1ll << 30)) return av2x::fail("%s: %lld x %d x %d (k a multiple of 32, n of 4)", what, (long long)rows, n, k);
    const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)((n + 63) / 64));
    if (w_is_kn) act8_gemm_kernel<true><<<grid, 256, 0, av2x::as_stream(stream)>>>(a, w, bias, residual, y, (int)rows, n, k);
    else act8_gemm_kernel<false><<<grid, 256, 0, av2x::as_stream(stream)>>>(a, w, bias, residual, y, (int)rows, n, k);
    return av2x::check_launch(what);
}
