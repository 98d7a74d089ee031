// Norms over the features of a row, alone and fused with what follows a block.
//
//   N(x) = (x - mu) s,  mu = mean(x) (0 for the RMS kind),  s = 1 / sqrt(mean((x - mu)^2) + eps)
//   norm            y = gamma N(x) + beta
//   gated residual  out = scale res + act(gate) gamma N(u)        and, on request,        y = gamma2 N2(out) + beta2
//
// Backward of the second from the gradients dout and dy, n = N(u), n2 = N2(out), q = act(gate):
//   a = dy gamma2;  d = dout + s2 (a - [mean a] - n2 mean(a n2));  dres = scale d;  dgate = d gamma n act'(gate)
//   b = d q gamma;  du = s (b - [mean b] - n mean(b n));  the means in brackets belong to the kind that subtracts one
//   dgamma = sum d q n,  dscale = sum d res,  dgamma2 = sum dy n2,  dbeta2 = sum dy over the rows
//
// What bounds it: the bytes, each tensor once.  A row stays in the registers of the G threads that share it, so that neither its moments nor
// the second norm read it again: forward 20 bytes an element (u, gate, res; out, y), backward 32 (dout, dy, u, gate, res; du, dgate,
// dres); out and its normalised values are formed anew in the backward from what it reads anyway.  Means and squares in two steps over the
// registers (first the mean, then the differences to it), sums in fp32 by halves.
// Sums over the rows: a thread always has the same columns, so it adds up its part in shared memory without a barrier; a block writes its
// sums once, and a last launch adds the blocks' in a fixed order: the same bits on every run.
#include "common.cuh"
#include "internal.h"
#include <initializer_list>
#include <type_traits>

namespace seera {

namespace {
constexpr int MAX_C = 8192;                    // features of a row: 64 floats a thread of 128, 16 of 512

// A row's threads and what each holds: V floats at column (thread + k G) V for each k < K.
template <int V> struct Piece { float x[V]; };
template <int V> __device__ __forceinline__ Piece<V> load(const float *p);
template <> __device__ __forceinline__ Piece<4> load<4>(const float *p) { const float4 v = *reinterpret_cast<const float4 *>(p); return {v.x, v.y, v.z, v.w}; }
template <> __device__ __forceinline__ Piece<1> load<1>(const float *p) { return {*p}; }
template <int V> __device__ __forceinline__ void store(float *p, const Piece<V> &v);
template <> __device__ __forceinline__ void store<4>(float *p, const Piece<4> &v) { *reinterpret_cast<float4 *>(p) = make_float4(v.x[0], v.x[1], v.x[2], v.x[3]); }
template <> __device__ __forceinline__ void store<1>(float *p, const Piece<1> &v) { *p = v.x[0]; }

// Both sums over the G threads of a row; `buf` alternates between two parts of the shared memory, so one barrier a call is enough.
template <int G> __device__ __forceinline__ float2 row_sum(float2 v, float2 (*sm)[32], int &buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
    if (G > 32) {
        if ((threadIdx.x & 31) == 0) sm[buf][threadIdx.x >> 5] = v;
        __syncthreads();
        v = sm[buf][0];
#pragma unroll
        for (int i = 1; i < G / 32; i++) { const float2 o = sm[buf][i]; v.x += o.x; v.y += o.y; }
        buf ^= 1;
    }
    return v;
}

// sigmoid(x) and 1 - sigmoid(x), both to full relative precision
__device__ __forceinline__ void sigmoid2(float x, float &p, float &q) {
    const float e = expf(-fabsf(x)), r = 1.f / (1.f + e);
    p = x >= 0.f ? r : e * r;
    q = x >= 0.f ? e * r : r;
    if (x != x) p = q = x;
}
__device__ __forceinline__ float gate_value(float g, int act) {
    float p, q;
    switch (act) {
        case SEERA_ACT_NONE: return g;
        case SEERA_ACT_RELU: return g > 0.f ? g : 0.f;
        case SEERA_ACT_TANH: return tanhf(g);
        default: sigmoid2(g, p, q); return act == SEERA_ACT_SIGMOID ? p : g * p;
    }
}
__device__ __forceinline__ float gate_slope(float g, int act, float &value) {
    float p, q;
    switch (act) {
        case SEERA_ACT_NONE: value = g; return 1.f;
        case SEERA_ACT_RELU: value = g > 0.f ? g : 0.f; return g > 0.f ? 1.f : 0.f;
        case SEERA_ACT_TANH: value = tanhf(g); return 1.f - value * value;
        default:
            sigmoid2(g, p, q);
            if (act == SEERA_ACT_SIGMOID) { value = p; return p * q; }
            value = g * p;
            return p * (1.f + g * q);
    }
}

// Moments of a row that its threads hold.
template <int G, int K, int V> __device__ __forceinline__ float2 moments(const Piece<V> (&x)[K], int C, int kind, float eps, int t, float2 (*sm)[32],
                                                                        int &buf) {
    const float inv = 1.f / (float)C;
    float mu = 0.f;
    if (kind == SEERA_NORM_LAYER) {
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < V; j++) s.x += x[k].x[j];      // (places behind the row hold zeros)
        mu = row_sum<G>(s, sm, buf).x * inv;
    }
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; k++)
        if ((t + k * G) * V < C) {
#pragma unroll
            for (int j = 0; j < V; j++) { const float d = x[k].x[j] - mu; s.x += d * d; }
        }
    return make_float2(mu, 1.f / sqrtf(row_sum<G>(s, sm, buf).x * inv + eps));
}

struct NormFwd {
    const float *x, *gamma, *beta;
    float *y, *stats;
    int rows, C, kind;
    float eps;
};
template <int G, int K, int V> __global__ void __launch_bounds__(G == 32 ? 256 : G) norm_fwd_kernel(const __grid_constant__ NormFwd p) {
    __shared__ float2 sm[2][32];
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, R = G == 32 ? 8 : 1;
    for (int row = blockIdx.x * R + (G == 32 ? threadIdx.x >> 5 : 0); row < p.rows; row += gridDim.x * R) {
        const long long at = (long long)row * p.C;
        Piece<V> x[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c < p.C) x[k] = load<V>(p.x + at + c);
            else x[k] = {};
        }
        const float2 ms = moments<G, K, V>(x, p.C, p.kind, p.eps, t, sm, buf);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
            const Piece<V> g = load<V>(p.gamma + c);
            Piece<V> o;
#pragma unroll
            for (int j = 0; j < V; j++) o.x[j] = (x[k].x[j] - ms.x) * ms.y * g.x[j];
            if (p.beta) {
                const Piece<V> b = load<V>(p.beta + c);
#pragma unroll
                for (int j = 0; j < V; j++) o.x[j] += b.x[j];
            }
            store<V>(p.y + at + c, o);
        }
        if (p.stats && t == 0) *reinterpret_cast<float2 *>(p.stats + 2ll * row) = ms;
    }
}

struct NormBwd {
    const float *dy, *x, *gamma, *stats;
    float *dx, *partial;
    int rows, C, kind;
};
template <int G, int K, int V> __global__ void __launch_bounds__(G == 32 ? 256 : G) norm_bwd_kernel(const __grid_constant__ NormBwd p) {
    __shared__ float2 sm[2][32];
    extern __shared__ float acc[];                         // [rows side by side][dgamma, dbeta][C]
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, R = G == 32 ? 8 : 1, lane_row = G == 32 ? threadIdx.x >> 5 : 0;
    float *mine = acc + (size_t)lane_row * 2 * p.C;
    for (int k = 0; k < K; k++) {
        const int c = (t + k * G) * V;
        if (c < p.C) { store<V>(mine + c, Piece<V>{}); store<V>(mine + p.C + c, Piece<V>{}); }
    }
    const float inv = 1.f / (float)p.C;
    for (int row = blockIdx.x * R + lane_row; row < p.rows; row += gridDim.x * R) {
        const long long at = (long long)row * p.C;
        const float2 ms = *reinterpret_cast<const float2 *>(p.stats + 2ll * row);
        Piece<V> n[K], d[K];
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c < p.C) { n[k] = load<V>(p.x + at + c); d[k] = load<V>(p.dy + at + c); }
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
            const Piece<V> g = load<V>(p.gamma + c);
            Piece<V> sg = load<V>(mine + c), sb = load<V>(mine + p.C + c);
#pragma unroll
            for (int j = 0; j < V; j++) {
                n[k].x[j] = (n[k].x[j] - ms.x) * ms.y;
                sg.x[j] += d[k].x[j] * n[k].x[j];
                sb.x[j] += d[k].x[j];
                d[k].x[j] *= g.x[j];
                s.x += d[k].x[j]; s.y += d[k].x[j] * n[k].x[j];
            }
            store<V>(mine + c, sg); store<V>(mine + p.C + c, sb);
        }
        s = row_sum<G>(s, sm, buf);
        const float m0 = p.kind == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C || !p.dx) break;
            Piece<V> o;
#pragma unroll
            for (int j = 0; j < V; j++) o.x[j] = ms.y * (d[k].x[j] - m0 - n[k].x[j] * m1);
            store<V>(p.dx + at + c, o);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.C; c += blockDim.x) {
        float r = acc[c];
        for (int i = 1; i < R; i++) r += acc[(size_t)i * 2 * p.C + c];
        p.partial[(size_t)blockIdx.x * 2 * p.C + c] = r;
    }
}

struct ResidualFwd {
    const float *u, *gate, *res, *gamma, *scale, *gamma2, *beta2;
    float *out, *y, *stats;
    long long ld_gate;
    int rows, C, kind, act, kind2;
    float eps, eps2;
};
template <int G, int K, int V> __global__ void __launch_bounds__(G == 32 ? 256 : G) residual_fwd_kernel(const __grid_constant__ ResidualFwd p) {
    __shared__ float2 sm[2][32];
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, R = G == 32 ? 8 : 1;
    for (int row = blockIdx.x * R + (G == 32 ? threadIdx.x >> 5 : 0); row < p.rows; row += gridDim.x * R) {
        const long long at = (long long)row * p.C;
        Piece<V> x[K], q[K], r[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            x[k] = {};
            if (c < p.C) {
                x[k] = load<V>(p.u + at + c);
                if (p.gate) q[k] = load<V>(p.gate + row * p.ld_gate + c);
                if (p.res) r[k] = load<V>(p.res + at + c);
            }
        }
        const float2 ms = moments<G, K, V>(x, p.C, p.kind, p.eps, t, sm, buf);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
            const Piece<V> g = load<V>(p.gamma + c);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float o = (x[k].x[j] - ms.x) * ms.y * g.x[j];
                if (p.gate) o *= gate_value(q[k].x[j], p.act);
                x[k].x[j] = o;
            }
            if (p.res) {
                const Piece<V> s = load<V>(p.scale + c);
#pragma unroll
                for (int j = 0; j < V; j++) x[k].x[j] += s.x[j] * r[k].x[j];
            }
            if (p.out) store<V>(p.out + at + c, x[k]);
        }
        float2 ms2 = {0.f, 0.f};
        if (p.y) {
            ms2 = moments<G, K, V>(x, p.C, p.kind2, p.eps2, t, sm, buf);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (t + k * G) * V;
                if (c >= p.C) break;
                const Piece<V> g = load<V>(p.gamma2 + c);
                Piece<V> o;
#pragma unroll
                for (int j = 0; j < V; j++) o.x[j] = (x[k].x[j] - ms2.x) * ms2.y * g.x[j];
                if (p.beta2) {
                    const Piece<V> b = load<V>(p.beta2 + c);
#pragma unroll
                    for (int j = 0; j < V; j++) o.x[j] += b.x[j];
                }
                store<V>(p.y + at + c, o);
            }
        }
        if (p.stats && t == 0) {
            float2 *st = reinterpret_cast<float2 *>(p.stats + 4ll * row);
            st[0] = ms;
            st[1] = ms2;
        }
    }
}

struct ResidualBwd {
    const float *dout, *dy, *u, *gate, *res, *gamma, *scale, *gamma2, *stats;
    float *du, *dgate, *dres, *partial;
    long long ld_gate, ld_dgate;
    int rows, C, kind, act, kind2;
};
template <int G, int K, int V> __global__ void __launch_bounds__(G == 32 ? 256 : G) residual_bwd_kernel(const __grid_constant__ ResidualBwd p) {
    __shared__ float2 sm[2][32];
    extern __shared__ float acc[];                         // [rows side by side][dgamma, dscale, dgamma2, dbeta2][C], the last two with dy
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, R = G == 32 ? 8 : 1, lane_row = G == 32 ? threadIdx.x >> 5 : 0;
    const int sums = p.dy ? 4 : 2;
    float *mine = acc + (size_t)lane_row * sums * p.C;
    for (int k = 0; k < K; k++) {
        const int c = (t + k * G) * V;
        if (c < p.C) for (int s = 0; s < sums; s++) store<V>(mine + s * p.C + c, Piece<V>{});
    }
    const float inv = 1.f / (float)p.C;
    for (int row = blockIdx.x * R + lane_row; row < p.rows; row += gridDim.x * R) {
        const long long at = (long long)row * p.C;
        const float4 st = *reinterpret_cast<const float4 *>(p.stats + 4ll * row);        // mu, s, mu2, s2
        Piece<V> n[K], g[K], r[K], d[K], e[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            d[k] = {};
            if (c < p.C) {
                n[k] = load<V>(p.u + at + c);
                if (p.gate) g[k] = load<V>(p.gate + row * p.ld_gate + c);
                if (p.res) r[k] = load<V>(p.res + at + c);
                if (p.dout) d[k] = load<V>(p.dout + at + c);
                if (p.dy) e[k] = load<V>(p.dy + at + c);
            }
        }
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
#pragma unroll
            for (int j = 0; j < V; j++) n[k].x[j] = (n[k].x[j] - st.x) * st.y;
        }
        if (p.dy) {
            Piece<V> n2[K];
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (t + k * G) * V;
                if (c >= p.C) break;
                const Piece<V> ga = load<V>(p.gamma + c), g2 = load<V>(p.gamma2 + c);
                Piece<V> sc = {}, sg = load<V>(mine + 2 * p.C + c), sb = load<V>(mine + 3 * p.C + c);
                if (p.res) sc = load<V>(p.scale + c);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float o = n[k].x[j] * ga.x[j];
                    if (p.gate) o *= gate_value(g[k].x[j], p.act);
                    if (p.res) o += sc.x[j] * r[k].x[j];
                    n2[k].x[j] = (o - st.z) * st.w;
                    sg.x[j] += e[k].x[j] * n2[k].x[j];
                    sb.x[j] += e[k].x[j];
                    e[k].x[j] *= g2.x[j];
                    s.x += e[k].x[j]; s.y += e[k].x[j] * n2[k].x[j];
                }
                store<V>(mine + 2 * p.C + c, sg); store<V>(mine + 3 * p.C + c, sb);
            }
            s = row_sum<G>(s, sm, buf);
            const float m0 = p.kind2 == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if ((t + k * G) * V >= p.C) break;
#pragma unroll
                for (int j = 0; j < V; j++) d[k].x[j] += st.w * (e[k].x[j] - m0 - n2[k].x[j] * m1);
            }
            s = {0.f, 0.f};
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
            const Piece<V> ga = load<V>(p.gamma + c);
            Piece<V> sg = load<V>(mine + c);
            if (p.res) {
                const Piece<V> sc = load<V>(p.scale + c);
                Piece<V> ss = load<V>(mine + p.C + c), o;
#pragma unroll
                for (int j = 0; j < V; j++) { ss.x[j] += d[k].x[j] * r[k].x[j]; o.x[j] = sc.x[j] * d[k].x[j]; }
                store<V>(mine + p.C + c, ss);
                if (p.dres) store<V>(p.dres + at + c, o);
            }
            if (p.gate) {
                Piece<V> o;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float q;
                    const float slope = gate_slope(g[k].x[j], p.act, q);
                    o.x[j] = d[k].x[j] * (ga.x[j] * n[k].x[j]) * slope;
                    d[k].x[j] *= q;
                }
                if (p.dgate) store<V>(p.dgate + row * p.ld_dgate + c, o);
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                sg.x[j] += d[k].x[j] * n[k].x[j];
                d[k].x[j] *= ga.x[j];
                s.x += d[k].x[j]; s.y += d[k].x[j] * n[k].x[j];
            }
            store<V>(mine + c, sg);
        }
        s = row_sum<G>(s, sm, buf);
        const float m0 = p.kind == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C || !p.du) break;
            Piece<V> o;
#pragma unroll
            for (int j = 0; j < V; j++) o.x[j] = st.y * (d[k].x[j] - m0 - n[k].x[j] * m1);
            store<V>(p.du + at + c, o);
        }
    }
    __syncthreads();
    const int all = sums * p.C;
    for (int c = threadIdx.x; c < all; c += blockDim.x) {
        float r = acc[c];
        for (int i = 1; i < R; i++) r += acc[(size_t)i * all + c];
        p.partial[(size_t)blockIdx.x * all + c] = r;
    }
}

// The blocks' sums added up in a fixed order, each of the up to four results to a place of its own (null: not wanted).
struct ParamSums { float *out[4]; };
__global__ void __launch_bounds__(1024) param_sums_kernel(const float *__restrict__ partial, const __grid_constant__ ParamSums to, int C, int n, int blocks) {
    __shared__ float sm[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, c = blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < n)
        for (int s = warp; s < blocks; s += 8 * warps) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = s + k * warps < blocks ? __ldg(partial + (size_t)(s + k * warps) * n + c) : 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) t += v[k];
        }
    sm[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && c < n) {
        float r = sm[0][lane];
        for (int w = 1; w < warps; w++) r += sm[w][lane];
        float *out = to.out[c / C];
        if (out) out[c % C] = r;
    }
}
int param_sums(const float *partial, const ParamSums &to, int C, int sums, int blocks, const char *name) {
    const int n = sums * C, threads = blocks <= 64 ? 256 : (blocks <= 128 ? 512 : 1024);
    param_sums_kernel<<<(n + 31) / 32, threads, 0, rt().stream>>>(partial, to, C, n, blocks);
    SEERA_LAUNCH_CHECK(name);
    return SEERA_OK;
}

template <int I> using Int = std::integral_constant<int, I>;
// The threads of a row: the fewest that hold it in at most 16 floats of each tensor.
template <class Fn> int by_width(int C, bool vec, Fn fn) {
    if (vec) {
        if (C <= 128) return fn(Int<32>{}, Int<1>{}, Int<4>{});
        if (C <= 256) return fn(Int<32>{}, Int<2>{}, Int<4>{});
        if (C <= 512) return fn(Int<128>{}, Int<1>{}, Int<4>{});
        if (C <= 1024) return fn(Int<128>{}, Int<2>{}, Int<4>{});
        if (C <= 2048) return fn(Int<256>{}, Int<2>{}, Int<4>{});
        if (C <= 4096) return fn(Int<512>{}, Int<2>{}, Int<4>{});
        return fn(Int<512>{}, Int<4>{}, Int<4>{});
    }
    if (C <= 128) return fn(Int<32>{}, Int<4>{}, Int<1>{});
    if (C <= 256) return fn(Int<32>{}, Int<8>{}, Int<1>{});
    if (C <= 512) return fn(Int<128>{}, Int<4>{}, Int<1>{});
    if (C <= 1024) return fn(Int<128>{}, Int<8>{}, Int<1>{});
    if (C <= 2048) return fn(Int<256>{}, Int<8>{}, Int<1>{});
    if (C <= 4096) return fn(Int<512>{}, Int<8>{}, Int<1>{});
    return fn(Int<512>{}, Int<16>{}, Int<1>{});
}
// Blocks of a launch that keeps sums over the rows: as many as are resident at once, so that each writes its sums once.
int resident_grid(const void *kernel, int threads, size_t smem, int rows, int rows_at_once, int *grid) {
    int per_sm = 0;
    if (int s = check_cuda(allow_smem(kernel, smem), "norm: shared memory")) return s;
    if (int s = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem), "norm: occupancy")) return s;
    const long long need = (rows + rows_at_once - 1) / rows_at_once, most = (long long)rt().sm_count * (per_sm > 0 ? per_sm : 1);
    *grid = (int)(need < most ? need : most);
    return SEERA_OK;
}
bool all16(std::initializer_list<const void *> ps) {
    for (const void *p : ps) if (!aligned16(p)) return false;
    return true;
}
bool norm_kind(int k) { return k == SEERA_NORM_RMS || k == SEERA_NORM_LAYER; }
}  // namespace

}  // namespace seera

using namespace seera;

extern "C" {

int seera_norm_fwd(const float *x, const float *gamma, const float *beta, float *y, float *stats, int rows, int C, int kind, float eps) {
    SEERA_ENSURE();
    if (rows < 0 || C < 1 || !norm_kind(kind) || !(eps >= 0.f) || (rows > 0 && (!x || !gamma || !y)) || ((uintptr_t)stats & 7))
        return fail(SEERA_E_ARG, "norm_fwd: bad argument");
    if (C > MAX_C) return fail(SEERA_E_LIMIT, "norm_fwd: %d features, at most %d", C, MAX_C);
    if (rows == 0) return SEERA_OK;
    const NormFwd p{x, gamma, beta, y, stats, rows, C, kind, eps};
    ProfBytes pb(8.0 * rows * C, "norm_fwd");
    return by_width(C, C % 4 == 0 && all16({x, gamma, beta, y}), [&](auto g_, auto k_, auto v_) {
        constexpr int G = decltype(g_)::value, K = decltype(k_)::value, V = decltype(v_)::value;
        norm_fwd_kernel<G, K, V><<<G == 32 ? (rows + 7) / 8 : rows, G == 32 ? 256 : G, 0, rt().stream>>>(p);
        SEERA_LAUNCH_CHECK("norm_fwd");
        return (int)SEERA_OK;
    });
}

int seera_norm_bwd(const float *dy, const float *x, const float *gamma, const float *stats, float *dx, float *dgamma, float *dbeta, int rows, int C,
                   int kind) {
    SEERA_ENSURE();
    if (rows < 1 || C < 1 || !norm_kind(kind) || !dy || !x || !gamma || !stats || ((uintptr_t)stats & 7))
        return fail(SEERA_E_ARG, "norm_bwd: bad argument");
    if (C > MAX_C) return fail(SEERA_E_LIMIT, "norm_bwd: %d features, at most %d", C, MAX_C);
    ProfBytes pb(12.0 * rows * C, "norm_bwd");
    return by_width(C, C % 4 == 0 && all16({dy, x, gamma, dx}), [&](auto g_, auto k_, auto v_) {
        constexpr int G = decltype(g_)::value, K = decltype(k_)::value, V = decltype(v_)::value;
        const int R = G == 32 ? 8 : 1, threads = G == 32 ? 256 : G;
        const size_t smem = (size_t)R * 2 * C * sizeof(float);
        int grid;
        if (int s = resident_grid((const void *)norm_bwd_kernel<G, K, V>, threads, smem, rows, R, &grid)) return s;
        float *partial = (float *)scratch_alloc((size_t)grid * 2 * C * sizeof(float));
        if (!partial) return (int)SEERA_E_OOM;
        const NormBwd p{dy, x, gamma, stats, dx, partial, rows, C, kind};
        norm_bwd_kernel<G, K, V><<<grid, threads, smem, rt().stream>>>(p);
        count_launch();
        int s = check_cuda(cudaGetLastError(), "norm_bwd");
        if (!s) s = param_sums(partial, {{dgamma, dbeta, nullptr, nullptr}}, C, 2, grid, "norm_bwd(sums)");
        scratch_free(partial);
        return s;
    });
}

int seera_gated_residual_fwd(const float *u, const float *gate, int ld_gate, const float *res, const float *gamma, const float *scale, float *out,
                             const float *next_gamma, const float *next_beta, float *y, float *stats, int rows, int C, int kind, int act,
                             int next_kind, float eps, float next_eps) {
    SEERA_ENSURE();
    if (rows < 0 || C < 1 || !norm_kind(kind) || act < SEERA_ACT_NONE || act > SEERA_ACT_SILU || !(eps >= 0.f) || (gate && ld_gate < C) ||
        (rows > 0 && (!u || !gamma || (!out && !y) || (res && !scale))) || (y && (!next_gamma || !norm_kind(next_kind) || !(next_eps >= 0.f))) ||
        ((uintptr_t)stats & 15))
        return fail(SEERA_E_ARG, "gated_residual_fwd: bad argument");
    if (C > MAX_C) return fail(SEERA_E_LIMIT, "gated_residual_fwd: %d features, at most %d", C, MAX_C);
    if (rows == 0) return SEERA_OK;
    const ResidualFwd p{u, gate, res, gamma, scale, next_gamma, next_beta, out, y, stats, ld_gate, rows, C, kind, act, next_kind, eps, next_eps};
    ProfBytes pb(4.0 * rows * C * (1 + (gate != nullptr) + (res != nullptr) + (out != nullptr) + (y != nullptr)), "gated_residual_fwd");
    const bool vec = C % 4 == 0 && (!gate || ld_gate % 4 == 0) && all16({u, gate, res, gamma, res ? scale : nullptr, out, y, y ? next_gamma : nullptr, y ? next_beta : nullptr});
    return by_width(C, vec, [&](auto g_, auto k_, auto v_) {
        constexpr int G = decltype(g_)::value, K = decltype(k_)::value, V = decltype(v_)::value;
        residual_fwd_kernel<G, K, V><<<G == 32 ? (rows + 7) / 8 : rows, G == 32 ? 256 : G, 0, rt().stream>>>(p);
        SEERA_LAUNCH_CHECK("gated_residual_fwd");
        return (int)SEERA_OK;
    });
}

int seera_gated_residual_bwd(const float *dout, const float *dy, const float *u, const float *gate, int ld_gate, const float *res, const float *gamma,
                             const float *scale, const float *next_gamma, const float *stats, float *du, float *dgate, int ld_dgate, float *dres,
                             float *dgamma, float *dscale, float *dnext_gamma, float *dnext_beta, int rows, int C, int kind, int act,
                             int next_kind) {
    SEERA_ENSURE();
    if (rows < 1 || C < 1 || !norm_kind(kind) || act < SEERA_ACT_NONE || act > SEERA_ACT_SILU || !u || !gamma || !stats || (!dout && !dy) ||
        (gate && ld_gate < C) || (dgate && (!gate || ld_dgate < C)) || (res && !scale) || ((dres || dscale) && !res) ||
        (dy && (!next_gamma || !norm_kind(next_kind))) || (!dy && (dnext_gamma || dnext_beta)) || ((uintptr_t)stats & 15))
        return fail(SEERA_E_ARG, "gated_residual_bwd: bad argument");
    if (C > MAX_C) return fail(SEERA_E_LIMIT, "gated_residual_bwd: %d features, at most %d", C, MAX_C);
    ProfBytes pb(4.0 * rows * C * (1 + (gate != nullptr) + (res != nullptr) + (dout != nullptr) + (dy != nullptr) + (du != nullptr) + (dgate != nullptr) +
                                   (dres != nullptr)), "gated_residual_bwd");
    const bool vec = C % 4 == 0 && (!gate || ld_gate % 4 == 0) && (!dgate || ld_dgate % 4 == 0) &&
                     all16({dout, dy, u, gate, res, gamma, res ? scale : nullptr, dy ? next_gamma : nullptr, du, dgate, dres});
    const int sums = dy ? 4 : 2;
    return by_width(C, vec, [&](auto g_, auto k_, auto v_) {
        constexpr int G = decltype(g_)::value, K = decltype(k_)::value, V = decltype(v_)::value;
        const int R = G == 32 ? 8 : 1, threads = G == 32 ? 256 : G;
        const size_t smem = (size_t)R * sums * C * sizeof(float);
        int grid;
        if (int s = resident_grid((const void *)residual_bwd_kernel<G, K, V>, threads, smem, rows, R, &grid)) return s;
        float *partial = (float *)scratch_alloc((size_t)grid * sums * C * sizeof(float));
        if (!partial) return (int)SEERA_E_OOM;
        const ResidualBwd p{dout, dy, u, gate, res, gamma, scale, next_gamma, stats, du, dgate, dres, partial, ld_gate, ld_dgate, rows, C, kind, act, next_kind};
        residual_bwd_kernel<G, K, V><<<grid, threads, smem, rt().stream>>>(p);
        count_launch();
        int s = check_cuda(cudaGetLastError(), "gated_residual_bwd");
        if (!s) s = param_sums(partial, {{dgamma, dscale, dnext_gamma, dnext_beta}}, C, sums, grid, "gated_residual_bwd(sums)");
        scratch_free(partial);
        return s;
    });
}

}  // extern "C"
