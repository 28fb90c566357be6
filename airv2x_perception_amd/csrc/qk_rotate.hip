// RMS norm of queries and keys per head with the position rotation in the same pass, forward and backward.
//
//   n = x / sqrt(mean(x^2) + eps),  u = n * gamma,  (a, b) -> (a cos t - b sin t, b cos t + a sin t)  for the D / 2 pairs of a head,
//   t = 2 pi pos[axis(i)] freq[i]  (freq in turns per unit of position; pair i belongs to axis i / (D / 2 / axes))
//   backward: du = the opposite turn of dy, dgamma = sum du n, g = du gamma, dx = (g - n mean(g n)) / sqrt(mean(x^2) + eps)
//
// Bound by HBM: every element is read and written once (backward: x and dy read, dx written).  A head vector of D elements is spread
// over D / 8 lanes that hold both elements of their four pairs -- the rotation needs no exchange, the norm log2(D / 8) shuffles.  Angles:
// the product pos * freq and its whole part in fp64 (a position of 1e6 keeps its phase), cos / sin of the rest in fp32, once per token
// and pair in LDS for all its heads.
// Measured: 140800 tokens x (8 + 8) heads of 32 in fp32: forward 114 us (577 MB, 5.1 TB/s), backward with the values' gradient 230 us (1.15 GB, 5.0 TB/s; a large copy
// reaches 4.9); 35200 tokens in bf16: 18.6 us; one token 2.8 us.
#include "token_common.hpp"

namespace {

constexpr int kTurnLds = 2048;     // (cos, sin) pairs a workgroup holds: 16 KB
// Head vectors per group of lanes and step.  Forward (us at 1 / 2 / 4 / 8 / 16): 140800 x 16 heads of 32 fp32: 117 / 116 / 120 / 125 / 138; 35200 x 8 heads of 128: 57 / 54 / 56 / 62 / 70.
// Backward, whose steps have two barriers (forward + backward at 4 / 8 / 16): 378 / 369 / 395; 181 / 183 / 191.
constexpr int kFwdVectors = 2, kBwdVectors = 8;
constexpr int kBwdGroups = 2048;   // workgroups of the backward pass: rows of the dgamma partials (1024: 35200 tokens in bf16 8 us slower; 4096: no faster)

struct RotArgs {
    const void *x[2];              // q, k
    long long sr[2], sh[2];        // element strides of a token and of a head
    const float* gamma[2];
    const int32_t* pos;
    const double* freqs;
    void* y[2];                    // forward: outputs (contiguous).  backward: dx, strides below
    const void* dy[3];             // backward: gradients of the outputs (contiguous); dv (may be null)
    long long yr[2], yh[2];
    void* dv;                      // backward: where the values' gradient goes (null: there is none)
    long long vr, vh;
    float* partial;                // backward: (2, groups, D)
    long long rows;
    int heads[2], axes, tok;       // tok: tokens per workgroup step
    float eps;
};

template <int D>
__device__ __forceinline__ void turns_to_lds(const RotArgs& a, long long t0, int nt, f32x2* cs) {
    constexpr int P = D / 2;
    const int per = P / a.axes;
    for (int i = threadIdx.x; i < nt * P; i += 256) {
        const int t = i / P, p = i % P;
        const double turns = (double)a.pos[(t0 + t) * a.axes + p / per] * a.freqs[p];
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cs[i] = f32x2{c, s};
    }
}

// the eight elements of a lane: INTER pairs (0,1) (2,3) ..: eight neighbours; else four of each half of the head
template <typename T, int D, bool INTER> __device__ __forceinline__ void load8(const T* v, int sub, f32x4& a, f32x4& b) {
    if constexpr (INTER) {
        const f32x4 u = tok_load4(v + sub * 8), w = tok_load4(v + sub * 8 + 4);
        a = f32x4{u.x, u.z, w.x, w.z};
        b = f32x4{u.y, u.w, w.y, w.w};
    } else {
        a = tok_load4(v + sub * 4);
        b = tok_load4(v + D / 2 + sub * 4);
    }
}
template <typename T, int D, bool INTER> __device__ __forceinline__ void store8(T* v, int sub, f32x4 a, f32x4 b) {
    if constexpr (INTER) {
        tok_store4(v + sub * 8, f32x4{a.x, b.x, a.y, b.y});
        tok_store4(v + sub * 8 + 4, f32x4{a.z, b.z, a.w, b.w});
    } else {
        tok_store4(v + sub * 4, a);
        tok_store4(v + D / 2 + sub * 4, b);
    }
}

__device__ __forceinline__ float dot4(f32x4 a, f32x4 b) { return (a.x * b.x + a.y * b.y) + (a.z * b.z + a.w * b.w); }

template <int LPV> __device__ __forceinline__ float vec_sum(float s) {
#pragma unroll
    for (int o = 1; o < LPV; o <<= 1) s += __shfl_xor(s, o);
    return s;
}

template <typename T, int D, bool INTER>
__global__ __launch_bounds__(256) void qk_rotate_kernel(RotArgs a) {
    constexpr int LPV = D / 8, VPW = 256 / LPV;
    __shared__ f32x2 cs[kTurnLds];
    const long long t0 = (long long)blockIdx.x * a.tok;
    const int nt = (int)min((long long)a.tok, a.rows - t0);
    turns_to_lds<D>(a, t0, nt, cs);
    __syncthreads();
    const int sub = threadIdx.x % LPV, nv = a.heads[0] + a.heads[1];
    f32x4 ga[2], gb[2];
#pragma unroll
    for (int w = 0; w < 2; ++w)
        if (a.gamma[w]) load8<float, D, INTER>(a.gamma[w], sub, ga[w], gb[w]);
    for (int v = threadIdx.x / LPV; v < nt * nv; v += VPW) {       // lanes of one head vector stay together
        const int t = v / nv;
        int h = v - t * nv;
        const bool isk = h >= a.heads[0];
        if (isk) h -= a.heads[0];
        f32x4 p, q;
        load8<T, D, INTER>(static_cast<const T*>(a.x[isk]) + (t0 + t) * a.sr[isk] + h * a.sh[isk], sub, p, q);
        const float r = 1.0f / sqrtf(vec_sum<LPV>(dot4(p, p) + dot4(q, q)) / (float)D + a.eps);
        p *= r * (isk ? ga[1] : ga[0]);
        q *= r * (isk ? gb[1] : gb[0]);
        const f32x2* c = cs + t * (D / 2) + sub * 4;
        f32x4 u, w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = p[i] * c[i].x - q[i] * c[i].y;
            w[i] = q[i] * c[i].x + p[i] * c[i].y;
        }
        store8<T, D, INTER>(static_cast<T*>(a.y[isk]) + ((t0 + t) * a.heads[isk] + h) * D, sub, u, w);
    }
}

template <typename T, int D, bool INTER>
__global__ __launch_bounds__(256) void qk_rotate_backward_kernel(RotArgs a) {
    constexpr int LPV = D / 8, VPW = 256 / LPV;
    __shared__ f32x2 cs[kTurnLds];
    __shared__ float red[4][2][D];
    const int sub = threadIdx.x % LPV, hq = a.heads[0], hk = a.heads[1];
    const int nv = hq + hk + (a.dv ? hk : 0);
    f32x4 ga[2], gb[2], da[2], db[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        da[w] = db[w] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.gamma[w]) load8<float, D, INTER>(a.gamma[w], sub, ga[w], gb[w]);
    }
    for (long long t0 = (long long)blockIdx.x * a.tok; t0 < a.rows; t0 += (long long)gridDim.x * a.tok) {
        const int nt = (int)min((long long)a.tok, a.rows - t0);
        __syncthreads();
        turns_to_lds<D>(a, t0, nt, cs);
        __syncthreads();
        for (int v = threadIdx.x / LPV; v < nt * nv; v += VPW) {
            const int t = v / nv;
            int h = v - t * nv;
            const long long tok = t0 + t;
            f32x4 u, w;
            if (h >= hq + hk) {        // values: their gradient passes through into the buffer's
                h -= hq + hk;
                u = w = f32x4{0.f, 0.f, 0.f, 0.f};
                if (a.dy[2]) load8<T, D, false>(static_cast<const T*>(a.dy[2]) + (tok * hk + h) * D, sub, u, w);
                store8<T, D, false>(static_cast<T*>(a.dv) + tok * a.vr + h * a.vh, sub, u, w);
                continue;
            }
            const bool isk = h >= hq;
            if (isk) h -= hq;
            f32x4 p, q;
            load8<T, D, INTER>(static_cast<const T*>(a.x[isk]) + tok * a.sr[isk] + h * a.sh[isk], sub, p, q);
            u = w = f32x4{0.f, 0.f, 0.f, 0.f};
            if (a.dy[isk]) load8<T, D, INTER>(static_cast<const T*>(a.dy[isk]) + (tok * a.heads[isk] + h) * D, sub, u, w);
            const f32x2* c = cs + t * (D / 2) + sub * 4;
            f32x4 gu, gw;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gu[i] = u[i] * c[i].x + w[i] * c[i].y;
                gw[i] = w[i] * c[i].x - u[i] * c[i].y;
            }
            const float r = 1.0f / sqrtf(vec_sum<LPV>(dot4(p, p) + dot4(q, q)) / (float)D + a.eps);
            p *= r;
            q *= r;
            if (isk) { da[1] += gu * p; db[1] += gw * q; gu *= ga[1]; gw *= gb[1]; }
            else { da[0] += gu * p; db[0] += gw * q; gu *= ga[0]; gw *= gb[0]; }
            const float m = vec_sum<LPV>(dot4(gu, p) + dot4(gw, q)) / (float)D;
            store8<T, D, INTER>(static_cast<T*>(a.y[isk]) + tok * a.yr[isk] + h * a.yh[isk], sub, (gu - p * m) * r, (gw - q * m) * r);
        }
    }
    // lanes with the same channels, then the four waves: a fixed order
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float s = da[w][i], t = db[w][i];
#pragma unroll
            for (int o = LPV; o < 64; o <<= 1) { s += __shfl_xor(s, o); t += __shfl_xor(t, o); }
            if ((threadIdx.x & 63) < LPV) {
                red[threadIdx.x >> 6][w][INTER ? sub * 8 + 2 * i : sub * 4 + i] = s;
                red[threadIdx.x >> 6][w][INTER ? sub * 8 + 2 * i + 1 : D / 2 + sub * 4 + i] = t;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 256)
        a.partial[((size_t)(i / D) * gridDim.x + blockIdx.x) * D + i % D] = (red[0][i / D][i % D] + red[1][i / D][i % D]) + (red[2][i / D][i % D] + red[3][i / D][i % D]);
}

// One workgroup per (q | k, 16 channels): 64 threads a channel take every 64th row, four sums each (a single chain of loads and adds is
// bound by their latency: 42 us for 2048 groups with 16 threads a channel), then a tree over the 64.  A fixed order for a given number of groups.
__global__ __launch_bounds__(1024) void qk_rotate_dgamma_kernel(const float* __restrict__ partial, int groups, int d, float* dq, float* dk) {
    __shared__ float red[64][16];
    float* out = blockIdx.y ? dk : dq;
    if (!out) return;
    const int ch = threadIdx.x & 15, r = threadIdx.x >> 4, c = blockIdx.x * 16 + ch;
    const float* src = partial + (size_t)blockIdx.y * groups * d + c;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = r; i < groups; i += 256)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += i + 64 * j < groups ? src[(size_t)(i + 64 * j) * d] : 0.f;
    red[r][ch] = (s[0] + s[1]) + (s[2] + s[3]);
    for (int o = 32; o; o >>= 1) {
        __syncthreads();
        if (r < o) red[r][ch] += red[r + o][ch];
    }
    if (r == 0) out[c] = red[0][ch];
}

template <typename F> int rot_dim(int dim, bool inter, F&& f) {
    switch (dim) {
        case 16: return inter ? f(std::integral_constant<int, 16>{}, std::true_type{}) : f(std::integral_constant<int, 16>{}, std::false_type{});
        case 32: return inter ? f(std::integral_constant<int, 32>{}, std::true_type{}) : f(std::integral_constant<int, 32>{}, std::false_type{});
        case 64: return inter ? f(std::integral_constant<int, 64>{}, std::true_type{}) : f(std::integral_constant<int, 64>{}, std::false_type{});
        default: return inter ? f(std::integral_constant<int, 128>{}, std::true_type{}) : f(std::integral_constant<int, 128>{}, std::false_type{});
    }
}

int rot_check(const char* what, const void* const* ptrs, int n_ptrs, const int64_t* strides, int n_strides, int64_t rows, int32_t heads, int32_t kv_heads,
              int32_t dim, int32_t axes, int32_t dtype, const void* pos, const void* freqs) {
    if (dim != 16 && dim != 32 && dim != 64 && dim != 128) return av2x::fail("%s: dim %d is not 16, 32, 64 or 128", what, dim);
    if (dtype < 0 || dtype > 2) return av2x::fail("%s: dtype %d", what, dtype);
    if (heads < 1 || heads > 1024 || kv_heads < 0 || kv_heads > 1024) return av2x::fail("%s: heads %d, kv_heads %d", what, heads, kv_heads);
    if (axes < 1 || (dim / 2) % axes) return av2x::fail("%s: %d axes do not divide %d pairs", what, axes, dim / 2);
    if (rows < 0 || rows > (1ll << 40)) return av2x::fail("%s: rows %lld", what, (long long)rows);
    if (rows > 0 && (!pos || !freqs)) return av2x::fail("%s: positions and frequencies are needed", what);
    const size_t al = 4 * tok_size(dtype);
    for (int i = 0; i < n_ptrs; ++i)
        if (!tok_aligned(ptrs[i], al)) return av2x::fail("%s: tensors must be aligned to four elements", what);
    for (int i = 0; i < n_strides; ++i)
        if (strides[i] % 4) return av2x::fail("%s: strides must be multiples of four elements", what);
    return 0;
}

// Tokens of a workgroup's step: `vectors` head vectors per group of lanes, the angles of all its tokens in LDS; on short inputs fewer, until there are 512 workgroups
// (300 tokens: forward 3.7 us, 8.5 without; 8800: 8.0 and 10.4).
int rot_tokens(int64_t rows, int dim, int nv, int vectors) {
    const int per_step = 256 / (dim / 8);
    int tok = (vectors * per_step + nv - 1) / nv;
    if (tok > kTurnLds / (dim / 2)) tok = kTurnLds / (dim / 2);
    if (tok < 1) tok = 1;
    while (tok > 1 && (rows + tok - 1) / tok < 512) tok = (tok + 1) / 2;
    return tok;
}

}  // namespace

extern "C" int av2x_qk_norm_rotate(const void* q, const void* k, const int64_t* strides, const float* gamma_q, const float* gamma_k,
                                   const int32_t* positions, const double* freqs, void* out_q, void* out_k, int64_t rows, int32_t heads,
                                   int32_t kv_heads, int32_t dim, int32_t axes, int32_t interleaved, int32_t dtype, float eps, av2x_stream_t stream) {
    const void* ptrs[] = {q, k, out_q, out_k, gamma_q, gamma_k};
    if (int rc = rot_check("av2x_qk_norm_rotate", ptrs, 4, strides, 4, rows, heads, kv_heads, dim, axes, dtype, positions, freqs)) return rc;
    if (rows == 0) return 0;
    if (!q || !out_q || !gamma_q || (kv_heads && (!k || !out_k || !gamma_k))) return av2x::fail("av2x_qk_norm_rotate: null tensor");
    if (!tok_aligned(gamma_q, 16) || !tok_aligned(gamma_k, 16)) return av2x::fail("av2x_qk_norm_rotate: gamma must be aligned to 16 bytes");
    RotArgs a{};
    a.x[0] = q; a.x[1] = k; a.sr[0] = strides[0]; a.sh[0] = strides[1]; a.sr[1] = strides[2]; a.sh[1] = strides[3];
    a.gamma[0] = gamma_q; a.gamma[1] = gamma_k; a.pos = positions; a.freqs = freqs; a.y[0] = out_q; a.y[1] = out_k;
    a.rows = rows; a.heads[0] = heads; a.heads[1] = kv_heads; a.axes = axes; a.eps = eps;
    a.tok = rot_tokens(rows, dim, heads + kv_heads, kFwdVectors);
    const int64_t grid = (rows + a.tok - 1) / a.tok;
    if (grid > 0x7fffffff) return av2x::fail("av2x_qk_norm_rotate: too many tokens");
    return rot_dim(dim, interleaved != 0, [&](auto d, auto inter) {
        AV2X_TOK_DISPATCH(dtype, T, (qk_rotate_kernel<T, decltype(d)::value, decltype(inter)::value><<<(unsigned)grid, 256, 0, av2x::as_stream(stream)>>>(a)));
        return av2x::check_launch("av2x_qk_norm_rotate");
    });
}

extern "C" uint64_t av2x_qk_norm_rotate_backward_workspace_bytes(int32_t dim) { return (uint64_t)2 * kBwdGroups * (dim > 0 ? dim : 0) * 4; }

extern "C" int av2x_qk_norm_rotate_backward(const void* q, const void* k, const int64_t* strides, const float* gamma_q, const float* gamma_k,
                                            const int32_t* positions, const double* freqs, const void* dout_q, const void* dout_k, const void* dout_v,
                                            void* dq, void* dk, void* dv, const int64_t* dstrides, float* dgamma_q, float* dgamma_k, int64_t rows,
                                            int32_t heads, int32_t kv_heads, int32_t dim, int32_t axes, int32_t interleaved, int32_t dtype, float eps,
                                            void* workspace, av2x_stream_t stream) {
    const void* ptrs[] = {q, k, dout_q, dout_k, dout_v, dq, dk, dv};
    if (int rc = rot_check("av2x_qk_norm_rotate_backward", ptrs, 8, strides, 4, rows, heads, kv_heads, dim, axes, dtype, positions, freqs)) return rc;
    for (int i = 0; i < 6; ++i)
        if (dstrides[i] % 4) return av2x::fail("av2x_qk_norm_rotate_backward: strides must be multiples of four elements");
    if (!gamma_q || (kv_heads && !gamma_k) || !workspace || (rows > 0 && (!q || !dq || (kv_heads && (!k || !dk))))) return av2x::fail("av2x_qk_norm_rotate_backward: null tensor");
    if (!tok_aligned(gamma_q, 16) || !tok_aligned(gamma_k, 16)) return av2x::fail("av2x_qk_norm_rotate_backward: gamma must be aligned to 16 bytes");
    RotArgs a{};
    a.x[0] = q; a.x[1] = k; a.sr[0] = strides[0]; a.sh[0] = strides[1]; a.sr[1] = strides[2]; a.sh[1] = strides[3];
    a.gamma[0] = gamma_q; a.gamma[1] = gamma_k; a.pos = positions; a.freqs = freqs;
    a.dy[0] = dout_q; a.dy[1] = dout_k; a.dy[2] = dout_v;
    a.y[0] = dq; a.y[1] = dk; a.yr[0] = dstrides[0]; a.yh[0] = dstrides[1]; a.yr[1] = dstrides[2]; a.yh[1] = dstrides[3];
    a.dv = dv; a.vr = dstrides[4]; a.vh = dstrides[5];
    a.partial = static_cast<float*>(workspace);
    a.rows = rows; a.heads[0] = heads; a.heads[1] = kv_heads; a.axes = axes; a.eps = eps;
    a.tok = rot_tokens(rows, dim, heads + kv_heads, kBwdVectors);
    int64_t grid = (rows + a.tok - 1) / a.tok;
    if (grid > kBwdGroups) grid = kBwdGroups;
    if (grid < 1) grid = 1;                       // no tokens: the partials are zeros, and so are the gammas' gradients
    return rot_dim(dim, interleaved != 0, [&](auto d, auto inter) {
        AV2X_TOK_DISPATCH(dtype, T, (qk_rotate_backward_kernel<T, decltype(d)::value, decltype(inter)::value><<<(unsigned)grid, 256, 0, av2x::as_stream(stream)>>>(a)));
        if (int rc = av2x::check_launch("av2x_qk_norm_rotate_backward")) return rc;
        if (!dgamma_q && !dgamma_k) return 0;
        qk_rotate_dgamma_kernel<<<dim3(dim / 16, 2), 1024, 0, av2x::as_stream(stream)>>>(a.partial, (int)grid, dim, dgamma_q, dgamma_k);
        return av2x::check_launch("av2x_qk_norm_rotate_backward: dgamma");
    });
}
