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
// Sums over the rows: a thread always has the same columns, so it adds up its part in registers; a block writes its sums once, and a last launch adds
// the blocks' in a fixed order: the same bits on every run.
// The backward kernels and the plain norm run as many blocks as are resident, each with the next row on its way while it works on one: what is left
// to wait for are two sums over the block's threads a row.  Measured (fp32, inputs beyond L2): norm of 16384 x 1280 both ways 82 us, 6 of them for the sums over
// the blocks (5.4 TB/s in the backward kernel); residual of 16384 x 2048 119 us forward (5.6 TB/s) and 201 backward (5.3 TB/s), the same with the gate as a range of wider
// rows.  Loads straight into registers, two blocks an SM and sums in shared memory took 297 for the last.
#include "common.cuh"
#include "internal.h"
#include "sigmoid.cuh"
#include "tc_ptx.cuh"
#include <algorithm>
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
// Zeros behind a row's end.  Kernels that do not end at it go through all of a thread's pieces, so that the loads of one do not wait for whether another is
// there.  Measured at 16384 rows: norm backward, single words 104 us of 2047 (ending early 109), V = 4 54 of 1280 when it ends early (60 when not); residual backward, single words
// 313 of 2047 (393), V = 4 see ENDS; the forward kernels end early (154 against 186 us).
template <int V> __device__ __forceinline__ Piece<V> load_if(const float *p, bool there) { return there ? load<V>(p) : Piece<V>{}; }
template <int V> __device__ __forceinline__ void store(float *p, const Piece<V> &v);
template <> __device__ __forceinline__ void store<4>(float *p, const Piece<4> &v) { *reinterpret_cast<float4 *>(p) = make_float4(v.x[0], v.x[1], v.x[2], v.x[3]); }
template <> __device__ __forceinline__ void store<1>(float *p, const Piece<1> &v) { *p = v.x[0]; }

// Sums over the threads of a row, a warp or a block; `buf` alternates between two parts of the shared memory, so one barrier a call is enough.
// (The places of the up to 16 warps are read independently of one another, several at once; what lies behind the last warp's is not used.)
struct __align__(16) Sums { float2 v[2][16]; };
template <int G> __device__ __forceinline__ float2 row_sum(float2 v, Sums &sm, int &buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
    if (G > 32) {
        if ((threadIdx.x & 31) == 0) sm.v[buf][threadIdx.x >> 5] = v;
        __syncthreads();
        v = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; i += 2)
            if (i * 32 < G) {
                const float4 o = *reinterpret_cast<const float4 *>(&sm.v[buf][i]);
                const bool more = (i + 1) * 32 < G;
                v.x += o.x + (more ? o.z : 0.f); v.y += o.y + (more ? o.w : 0.f);
            }
        buf ^= 1;
    }
    return v;
}
template <int G> __device__ __forceinline__ float row_sum(float x, Sums &sm, int &buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (G > 32) {
        float *place = &sm.v[buf][0].x;
        if ((threadIdx.x & 31) == 0) place[threadIdx.x >> 5] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            if (i * 32 < G) {
                const float4 o = *reinterpret_cast<const float4 *>(place + i);
                const int left = G / 32 - i;
                x += (o.x + (left > 1 ? o.y : 0.f)) + ((left > 2 ? o.z : 0.f) + (left > 3 ? o.w : 0.f));
            }
        buf ^= 1;
    }
    return x;
}

// sigmoid(x) and 1 - sigmoid(x), both to full relative precision
__device__ __forceinline__ void sigmoid2(float x, float &p, float &q) {
    const float s = fabsf(sigmoid_less(x)), b = 1.f - s;
    p = x >= 0.f ? b : s;
    q = x >= 0.f ? s : b;
}
template <int K, int V, class Fn> __device__ __forceinline__ void each(Piece<V> (&g)[K], Fn fn) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int j = 0; j < V; j++) fn(k, j, g[k].x[j]);
}
// g -> act(g)
template <int K, int V> __device__ __forceinline__ void gate_values(Piece<V> (&g)[K], int act) {
    switch (act) {
        case SEERA_ACT_NONE: return;
        case SEERA_ACT_RELU: each<K, V>(g, [](int, int, float &x) { x = x > 0.f ? x : 0.f; }); return;
        case SEERA_ACT_TANH: each<K, V>(g, [](int, int, float &x) { x = tanhf(x); }); return;
        case SEERA_ACT_SIGMOID: each<K, V>(g, [](int, int, float &x) { float p, q; sigmoid2(x, p, q); x = p; }); return;
        default: each<K, V>(g, [](int, int, float &x) { float p, q; sigmoid2(x, p, q); x *= p; });
    }
}
// g -> act(g), with act'(g) beside it
template <int K, int V> __device__ __forceinline__ void gate_slopes(Piece<V> (&g)[K], Piece<V> (&slope)[K], int act) {
    switch (act) {
        case SEERA_ACT_NONE: each<K, V>(g, [&](int k, int j, float &) { slope[k].x[j] = 1.f; }); return;
        case SEERA_ACT_RELU: each<K, V>(g, [&](int k, int j, float &x) { slope[k].x[j] = x > 0.f ? 1.f : 0.f; x = x > 0.f ? x : 0.f; }); return;
        case SEERA_ACT_TANH: each<K, V>(g, [&](int k, int j, float &x) { x = tanhf(x); slope[k].x[j] = 1.f - x * x; }); return;
        case SEERA_ACT_SIGMOID: each<K, V>(g, [&](int k, int j, float &x) { float p, q; sigmoid2(x, p, q); slope[k].x[j] = p * q; x = p; }); return;
        default: each<K, V>(g, [&](int k, int j, float &x) { float p, q; sigmoid2(x, p, q); slope[k].x[j] = p * (1.f + x * q); x *= p; });
    }
}

// The rows of N tensors on their way to the thread that works on them, one row ahead: each thread copies what it will read itself, so that
// nothing has to be waited for but its own copies, and the loads hold no registers.  Rows of more than 8 floats a thread would not leave room for it.
// (A place of its own for each thread, at constant distances, took half as long again as the copies of a warp side by side.)
// Loads into registers instead, us of 16384 x 2048 / 2047: with one tensor 53 / 64 (here 51 / 75), with two 102 / 109 (77 / 103), with five 222 / 367 (203 / 313).
// With three, the forward of the residual, they are used: 113 / 141 (a row ahead: 115 / 209, the odd row's single copies and reads).
// Two rows ahead: 52, 81 and, with half the blocks, 300 us of 2048.
template <int K, int V> constexpr bool AHEAD = K * V <= 8;
template <int G, int K, int V, int N> struct Ahead {
    static constexpr bool ON = AHEAD<K, V> && N != 3;
    static constexpr int STAGES = 2;
    static constexpr int STAGE = N * K * V * G;
    static constexpr size_t FLOATS = ON ? STAGES * STAGE : 0;          // of a row
    float *mine, *asked;                                   // asked: the stage that is asked for next
    int t, C;
    Piece<V> now[ON ? 1 : N][ON ? 1 : K];
    __device__ __forceinline__ Ahead(float *mem, int t_, int C_) : mine(mem + (G == 32 ? (threadIdx.x >> 5) * FLOATS : 0) + t_ * V), asked(mine), t(t_), C(C_) {}
    __device__ __forceinline__ float *place(int i, int k) const { return asked + (i * K + k) * (G * V); }
    // a row of tensor i (null: zeros) is asked for; `next()` behind the last of them
    __device__ __forceinline__ void request(int i, const float *row) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if constexpr (ON) {
                if (!row || c >= C) continue;
                if (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(place(i, k))), "l"(row + c) : "memory");
                else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(place(i, k))), "l"(row + c) : "memory");
            } else {
                now[i][k] = {};
                if (row && c < C) now[i][k] = load<V>(row + c);
            }
        }
    }
    __device__ __forceinline__ void next() {
        if (!ON) return;
        asm volatile("cp.async.commit_group;" ::: "memory");
        asked = asked + STAGE == mine + STAGES * STAGE ? mine : asked + STAGE;
    }
    // The row that was asked for in front of the last STAGES - 1 calls of `next()` is there, in the stage that is asked for next; those asked for since may
    // still be on their way.
    __device__ __forceinline__ void wait() { if (ON) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
    __device__ __forceinline__ Piece<V> take(int i, int k, bool there) const {
        if constexpr (ON) return there && (t + k * G) * V < C ? load<V>(place(i, k)) : Piece<V>{};
        else return now[i][k];
    }
};

// Sums over the rows for the thread's columns, in registers where a row is short enough, else in shared memory.
template <int G, int K, int V> struct Sum {
    static constexpr bool ON = AHEAD<K, V>;
    Piece<V> r[ON ? K : 1];
    float *mem;
    int C;
    __device__ __forceinline__ Sum(float *mem_, int t, int C_) : mem(mem_), C(C_) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if constexpr (ON) r[k] = {};
            else if (c < C) store<V>(mem + c, Piece<V>{});
        }
    }
    template <class Fn> __device__ __forceinline__ void add(int k, int c, Fn what) {
        if constexpr (ON) {
#pragma unroll
            for (int j = 0; j < V; j++) r[k].x[j] += what(j);
        } else if (V > 1 || c < C) {
            Piece<V> s = load<V>(mem + c);
#pragma unroll
            for (int j = 0; j < V; j++) s.x[j] += what(j);
            store<V>(mem + c, s);
        }
    }
    __device__ __forceinline__ void keep(int t, int C) const {         // to shared memory
        if constexpr (ON) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (t + k * G) * V;
                if (c < C) store<V>(mem + c, r[k]);
            }
        }
    }
};

// Moments of a row that its threads hold.
template <int G, int K, int V> __device__ __forceinline__ float2 moments(const Piece<V> (&x)[K], int C, int kind, float eps, int t, Sums &sm,
                                                                           int &buf) {
    const float inv = 1.f / (float)C;
    float mu = 0.f;
    if (kind == SEERA_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < V; j++) s += x[k].x[j];        // (places behind the row hold zeros)
        mu = row_sum<G>(s, sm, buf) * inv;
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; k++)
        if ((t + k * G) * V < C) {
#pragma unroll
            for (int j = 0; j < V; j++) { const float d = x[k].x[j] - mu; s += d * d; }
        }
    return make_float2(mu, 1.f / sqrtf(row_sum<G>(s, sm, buf) * inv + eps));
}

struct NormFwd {
    const float *x, *gamma, *beta;
    float *y, *stats;
    int rows, C, kind;
    float eps;
};
// A block's threads, and its rows side by side.
template <int G> constexpr int THREADS_OF = G == 32 ? 256 : G;
template <int G> constexpr int ROWS_OF = G == 32 ? 8 : 1;

template <int G, int K, int V> __global__ void __launch_bounds__(THREADS_OF<G>, 1024 / THREADS_OF<G>) norm_fwd_kernel(const __grid_constant__ NormFwd p) {
    __shared__ Sums sm;
    extern __shared__ __align__(16) float mem[];
    typedef Ahead<G, K, V, 1> Rows;
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, side = G == 32 ? threadIdx.x >> 5 : 0, step = gridDim.x * ROWS_OF<G>;
    Rows in(mem, t, p.C);
    unsigned row = blockIdx.x * ROWS_OF<G> + side;      // (rows + 2 step passes 31 bits, not 32)
    auto request = [&](unsigned row) {
        if (row < p.rows) in.request(0, p.x + (long long)row * p.C);
        in.next();
    };
    if (Rows::ON)
        for (int k = 0; k < Rows::STAGES - 1; k++) request(row + k * step);
    for (; row < p.rows; row += step) {
        request(Rows::ON ? row + (Rows::STAGES - 1) * step : row);
        in.wait();
        const long long at = (long long)row * p.C;
        Piece<V> x[K];
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = in.take(0, k, true);
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

// A block's sums over its rows from shared memory [rows side by side][sums][C] to its place in global memory.
template <int G> __device__ __forceinline__ void write_sums(const float *acc, float *partial, int all) {
    __syncthreads();
    for (int c = threadIdx.x; c < all; c += blockDim.x) {
        float r = acc[c];
        for (int i = 1; i < ROWS_OF<G>; i++) r += acc[(size_t)i * all + c];
        partial[(size_t)blockIdx.x * all + c] = r;
    }
}

struct NormBwd {
    const float *dy, *x, *gamma, *stats;
    float *dx, *partial;
    int rows, C, kind;
};
template <int G, int K, int V> __global__ void __launch_bounds__(THREADS_OF<G>, 512 / THREADS_OF<G>) norm_bwd_kernel(const __grid_constant__ NormBwd p) {
    __shared__ Sums sm;
    extern __shared__ __align__(16) float mem[];           // rows on their way, then (or instead) [rows side by side][dgamma, dbeta][C]
    typedef Ahead<G, K, V, 2> Rows;
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, side = G == 32 ? threadIdx.x >> 5 : 0, step = gridDim.x * ROWS_OF<G>;
    float *acc = mem + (size_t)side * 2 * p.C;
    Sum<G, K, V> sg(acc, t, p.C), sb(acc + p.C, t, p.C);
    Rows in(mem, t, p.C);
    unsigned row = blockIdx.x * ROWS_OF<G> + side;      // (rows + 2 step passes 31 bits, not 32)
    auto request = [&](unsigned row) {
        if (row < p.rows) {
            in.request(0, p.x + (long long)row * p.C);
            in.request(1, p.dy + (long long)row * p.C);
        }
        in.next();
    };
    if (Rows::ON)
        for (int k = 0; k < Rows::STAGES - 1; k++) request(row + k * step);
    const float inv = 1.f / (float)p.C;
    auto stats = [&](unsigned row) { return row < p.rows ? *reinterpret_cast<const float2 *>(p.stats + 2ll * row) : float2{}; };
    float2 ms_next = stats(row);
    for (; row < p.rows; row += step) {
        const float2 ms = ms_next;
        ms_next = stats(row + step);
        request(Rows::ON ? row + (Rows::STAGES - 1) * step : row);
        in.wait();
        Piece<V> n[K], d[K];
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            n[k] = in.take(0, k, true);
            d[k] = in.take(1, k, true);
            if (V > 1 && c >= p.C) break;
            const Piece<V> g = load_if<V>(p.gamma + c, V > 1 || c < p.C);
#pragma unroll
            for (int j = 0; j < V; j++) n[k].x[j] = (n[k].x[j] - ms.x) * ms.y;
            sg.add(k, c, [&](int j) { return d[k].x[j] * n[k].x[j]; });
            sb.add(k, c, [&](int j) { return d[k].x[j]; });
#pragma unroll
            for (int j = 0; j < V; j++) {
                d[k].x[j] *= g.x[j];
                s.x += d[k].x[j]; s.y += d[k].x[j] * n[k].x[j];
            }
        }
        s = row_sum<G>(s, sm, buf);
        const float m0 = p.kind == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C || !p.dx) {
                if (V > 1) break;
                continue;
            }
            Piece<V> o;
#pragma unroll
            for (int j = 0; j < V; j++) o.x[j] = ms.y * (d[k].x[j] - m0 - n[k].x[j] * m1);
            store<V>(p.dx + (long long)row * p.C + c, o);
        }
    }
    __syncthreads();                                       // (the places of the rows are read)
    sg.keep(t, p.C); sb.keep(t, p.C);
    write_sums<G>(mem, p.partial, 2 * p.C);
}

struct ResidualFwd {
    const float *u, *gate, *res, *gamma, *scale, *gamma2, *beta2;
    float *out, *y, *stats;
    long long ld_gate;
    int rows, C, kind, act, kind2;
    float eps, eps2;
};
template <int G, int K, int V> __global__ void __launch_bounds__(THREADS_OF<G>, (AHEAD<K, V> ? 1024 : 512) / THREADS_OF<G>) residual_fwd_kernel(const __grid_constant__ ResidualFwd p) {
    __shared__ Sums sm;
    extern __shared__ __align__(16) float mem[];
    typedef Ahead<G, K, V, 3> Rows;
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, side = G == 32 ? threadIdx.x >> 5 : 0, step = gridDim.x * ROWS_OF<G>;
    Rows in(mem, t, p.C);
    unsigned row = blockIdx.x * ROWS_OF<G> + side;      // (rows + 2 step passes 31 bits, not 32)
    auto request = [&](unsigned row) {
        if (row < p.rows) {
            in.request(0, p.u + (long long)row * p.C);
            in.request(1, p.gate ? p.gate + row * p.ld_gate : nullptr);
            in.request(2, p.res ? p.res + (long long)row * p.C : nullptr);
        }
        in.next();
    };
    for (; row < p.rows; row += step) {
        request(row);
        const long long at = (long long)row * p.C;
        Piece<V> x[K], q[K], r[K];
#pragma unroll
        for (int k = 0; k < K; k++) { x[k] = in.take(0, k, true); q[k] = in.take(1, k, p.gate); r[k] = in.take(2, k, p.res); }
        const float2 ms = moments<G, K, V>(x, p.C, p.kind, p.eps, t, sm, buf);
        if (p.gate) gate_values<K, V>(q, p.act);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C) break;
            const Piece<V> g = load<V>(p.gamma + c);
#pragma unroll
            for (int j = 0; j < V; j++) x[k].x[j] = (x[k].x[j] - ms.x) * ms.y * g.x[j];
            if (p.gate) {
#pragma unroll
                for (int j = 0; j < V; j++) x[k].x[j] *= q[k].x[j];
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
template <int G, int K, int V> __global__ void __launch_bounds__(THREADS_OF<G>, 512 / THREADS_OF<G>) residual_bwd_kernel(const __grid_constant__ ResidualBwd p) {
    // Whether pieces behind a row's end are left out.  Going through them is faster where registers allow (16384 x 2048 194 against 203 us, x 1280 128 against 136,
    // x 768 82 against 85), not for rows of a warp (65536 x 256 104 against 99) and where it spills (8192 x 4096 271 against 231, x 3300 259 against 237).
    constexpr bool ENDS = V > 1 && (G == 32 || G > 320);
    __shared__ Sums sm;
    extern __shared__ __align__(16) float mem[];           // rows on their way, then (or instead) [rows side by side][dgamma, dscale, dgamma2, dbeta2][C],
    typedef Ahead<G, K, V, 5> Rows;                        // the last two with dy
    int buf = 0;
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, side = G == 32 ? threadIdx.x >> 5 : 0, step = gridDim.x * ROWS_OF<G>;
    const int sums = p.dy ? 4 : 2;
    float *acc = mem + (size_t)side * sums * p.C;
    Sum<G, K, V> sum_gamma(acc, t, p.C), sum_scale(acc + p.C, t, p.C), sum_gamma2(acc + (sums - 2) * p.C, t, p.C), sum_beta2(acc + (sums - 1) * p.C, t, p.C);
    Rows in(mem, t, p.C);
    unsigned row = blockIdx.x * ROWS_OF<G> + side;      // (rows + 2 step passes 31 bits, not 32)
    auto request = [&](unsigned row) {
        if (row < p.rows) {
            const long long at = (long long)row * p.C;
            in.request(0, p.u + at);
            in.request(1, p.gate ? p.gate + row * p.ld_gate : nullptr);
            in.request(2, p.res ? p.res + at : nullptr);
            in.request(3, p.dout ? p.dout + at : nullptr);
            in.request(4, p.dy ? p.dy + at : nullptr);
        }
        in.next();
    };
    if (Rows::ON)
        for (int k = 0; k < Rows::STAGES - 1; k++) request(row + k * step);
    const float inv = 1.f / (float)p.C;
    auto stats = [&](unsigned row) { return row < p.rows ? *reinterpret_cast<const float4 *>(p.stats + 4ll * row) : float4{}; };
    float4 st_next = stats(row);
    for (; row < p.rows; row += step) {
        const float4 st = st_next;                         // mu, s, mu2, s2
        st_next = stats(row + step);
        request(Rows::ON ? row + (Rows::STAGES - 1) * step : row);
        in.wait();
        const long long at = (long long)row * p.C;
        Piece<V> n[K], g[K], slope[Rows::ON ? K : 1], r[K], d[K];
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++) {
            n[k] = in.take(0, k, true);
#pragma unroll
            for (int j = 0; j < V; j++) n[k].x[j] = (n[k].x[j] - st.x) * st.y;
            g[k] = in.take(1, k, p.gate);
            r[k] = in.take(2, k, p.res);
            d[k] = in.take(3, k, p.dout);
        }
        // (a row of many floats a thread has no registers for values and slopes at once: they are formed where they are used)
        if constexpr (Rows::ON) { if (p.gate) gate_slopes<K, V>(g, slope, p.act); }
        if (p.dy) {
            Piece<V> n2[K], e[K];
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (t + k * G) * V;
                e[k] = in.take(4, k, true);
                if (ENDS && c >= p.C) break;
                const Piece<V> ga = load_if<V>(p.gamma + c, ENDS || c < p.C), g2 = load_if<V>(p.gamma2 + c, ENDS || c < p.C);
                Piece<V> sc = {}, q[1] = {g[k]};
                if (p.res) sc = load_if<V>(p.scale + c, ENDS || c < p.C);
                if (!Rows::ON && p.gate) gate_values<1, V>(q, p.act);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float o = n[k].x[j] * ga.x[j];
                    if (p.gate) o *= q[0].x[j];
                    if (p.res) o += sc.x[j] * r[k].x[j];
                    n2[k].x[j] = (o - st.z) * st.w;
                }
                sum_gamma2.add(k, c, [&](int j) { return e[k].x[j] * n2[k].x[j]; });
                sum_beta2.add(k, c, [&](int j) { return e[k].x[j]; });
#pragma unroll
                for (int j = 0; j < V; j++) {
                    e[k].x[j] *= g2.x[j];
                    s.x += e[k].x[j]; s.y += e[k].x[j] * n2[k].x[j];
                }
            }
            s = row_sum<G>(s, sm, buf);
            const float m0 = p.kind2 == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (ENDS && (t + k * G) * V >= p.C) break;
#pragma unroll
                for (int j = 0; j < V; j++) d[k].x[j] += st.w * (e[k].x[j] - m0 - n2[k].x[j] * m1);
            }
            s = {0.f, 0.f};
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (ENDS && c >= p.C) break;
            const Piece<V> ga = load_if<V>(p.gamma + c, ENDS || c < p.C);
            if (p.res) {
                const Piece<V> sc = load_if<V>(p.scale + c, ENDS || c < p.C);
                Piece<V> o;
                sum_scale.add(k, c, [&](int j) { return d[k].x[j] * r[k].x[j]; });
#pragma unroll
                for (int j = 0; j < V; j++) o.x[j] = sc.x[j] * d[k].x[j];
                if (p.dres && (ENDS || c < p.C)) store<V>(p.dres + at + c, o);
            }
            if (p.gate) {
                Piece<V> o, q[1] = {g[k]}, sl[1] = {slope[Rows::ON ? k : 0]};
                if (!Rows::ON) gate_slopes<1, V>(q, sl, p.act);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    o.x[j] = d[k].x[j] * (ga.x[j] * n[k].x[j]) * sl[0].x[j];
                    d[k].x[j] *= q[0].x[j];
                }
                if (p.dgate && (ENDS || c < p.C)) store<V>(p.dgate + row * p.ld_dgate + c, o);
            }
            sum_gamma.add(k, c, [&](int j) { return d[k].x[j] * n[k].x[j]; });
#pragma unroll
            for (int j = 0; j < V; j++) {
                d[k].x[j] *= ga.x[j];
                s.x += d[k].x[j]; s.y += d[k].x[j] * n[k].x[j];
            }
        }
        s = row_sum<G>(s, sm, buf);
        const float m0 = p.kind == SEERA_NORM_LAYER ? s.x * inv : 0.f, m1 = s.y * inv;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (t + k * G) * V;
            if (c >= p.C || !p.du) {
                if (ENDS) break;
                continue;
            }
            Piece<V> o;
#pragma unroll
            for (int j = 0; j < V; j++) o.x[j] = st.y * (d[k].x[j] - m0 - n[k].x[j] * m1);
            store<V>(p.du + at + c, o);
        }
    }
    __syncthreads();                                       // (the places of the rows are read)
    sum_gamma.keep(t, p.C); sum_scale.keep(t, p.C);
    if (p.dy) { sum_gamma2.keep(t, p.C); sum_beta2.keep(t, p.C); }
    write_sums<G>(mem, p.partial, sums * p.C);
}

// The blocks' sums added up in a fixed order, each of the up to four results to a place of its own (null: not wanted).
struct ParamSums { float *out[4]; };
// A block has 32 columns; its warps take the rows, V at a time in pieces of V columns a lane.  Measured: 296 blocks' sums of 8192 columns 7.1 us.
template <int V> __global__ void __launch_bounds__(1024) param_sums_kernel(const float *__restrict__ partial, const __grid_constant__ ParamSums to, int C, int n,
                                                                           int blocks) {
    constexpr int ACROSS = 32 / V, AT_ONCE = 4;
    __shared__ float sm[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, c = blockIdx.x * 32 + lane % ACROSS * V, step = warps * V;
    Piece<V> t = {};
    if (c < n)
        for (int s = warp * V + lane / ACROSS; s < blocks; s += AT_ONCE * step) {
            Piece<V> v[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) v[k] = s + k * step < blocks ? load<V>(partial + (size_t)(s + k * step) * n + c) : Piece<V>{};
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++)
#pragma unroll
                for (int j = 0; j < V; j++) t.x[j] += v[k].x[j];
        }
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
        for (int o = ACROSS; o < 32; o <<= 1) t.x[j] += __shfl_xor_sync(0xffffffffu, t.x[j], o);
        if (lane < ACROSS) sm[warp][lane * V + j] = t.x[j];
    }
    __syncthreads();
    for (int k = warp; k < 32; k += warps) {               // a warp adds up a column
        float r = lane < warps ? sm[lane][k] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
        const int at = blockIdx.x * 32 + k;
        if (lane == 0 && at < n && to.out[at / C]) to.out[at / C][at % C] = r;
    }
}
int param_sums(const float *partial, const ParamSums &to, int C, int sums, int blocks, const char *name) {
    const int n = sums * C, threads = blocks <= 64 ? 256 : (blocks <= 128 ? 512 : 1024);
    if (n % 4 == 0) param_sums_kernel<4><<<(n + 31) / 32, threads, 0, rt().stream>>>(partial, to, C, n, blocks);
    else param_sums_kernel<1><<<(n + 31) / 32, threads, 0, rt().stream>>>(partial, to, C, n, blocks);
    SEERA_LAUNCH_CHECK(name);
    return SEERA_OK;
}

template <int I> using Int = std::integral_constant<int, I>;
// The threads of a row: the fewest of these that hold it in 8 floats of each tensor, or 512 with 16; each at most a third more than the one before (from 96 on), since
// threads without work cost: of 16384 rows of 768 the residual's two directions take 48 and 85 us with 96 threads, 53 and 93 with 128; of 2560 147 and 308
// with 320, 205 and 365 with 512; of 1280 74 and 136 with 160, 82 and 148 with 192.
template <class Fn, class K, class V> int by_threads(int C, Fn fn, K k, V v) {
    const int threads = (C + 7) / 8;
    if (threads <= 32) return fn(Int<32>{}, k, v);
    if (threads <= 64) return fn(Int<64>{}, k, v);
    if (threads <= 96) return fn(Int<96>{}, k, v);
    if (threads <= 128) return fn(Int<128>{}, k, v);
    if (threads <= 160) return fn(Int<160>{}, k, v);
    if (threads <= 192) return fn(Int<192>{}, k, v);
    if (threads <= 256) return fn(Int<256>{}, k, v);
    if (threads <= 320) return fn(Int<320>{}, k, v);
    if (threads <= 416) return fn(Int<416>{}, k, v);
    return fn(Int<512>{}, k, v);
}
template <class Fn> int by_width(int C, bool vec, Fn fn) {
    if (C > 4096) return vec ? fn(Int<512>{}, Int<4>{}, Int<4>{}) : fn(Int<512>{}, Int<16>{}, Int<1>{});
    if (!vec && C <= 64) return fn(Int<32>{}, Int<2>{}, Int<1>{});
    return vec ? by_threads(C, fn, Int<2>{}, Int<4>{}) : by_threads(C, fn, Int<8>{}, Int<1>{});
}
// Blocks of a launch that keeps sums over the rows: as many as are resident at once, so that each writes its sums once.
// (`known` is the kernel's: asking takes the host longer than half a launch.)
struct PerSm { size_t smem = 0; int blocks = 0; };
int resident_grid(PerSm &known, const void *kernel, int threads, size_t smem, int rows, int rows_at_once, int *grid) {
    if (!known.blocks || known.smem != smem) {
        if (int s = check_cuda(allow_smem(kernel, smem), "norm: shared memory")) return s;
        if (int s = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&known.blocks, kernel, threads, smem), "norm: occupancy")) return s;
        known.smem = smem;
    }
    const long long need = ((long long)rows + rows_at_once - 1) / rows_at_once, most = (long long)rt().sm_count * (known.blocks > 0 ? known.blocks : 1);
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
        const size_t smem = ROWS_OF<G> * Ahead<G, K, V, 1>::FLOATS * sizeof(float);
        int grid = (int)(((long long)rows + ROWS_OF<G> - 1) / ROWS_OF<G>);
        static PerSm known;
        if (Ahead<G, K, V, 1>::ON) if (int s = resident_grid(known, (const void *)norm_fwd_kernel<G, K, V>, THREADS_OF<G>, smem, rows, ROWS_OF<G>, &grid)) return s;
        norm_fwd_kernel<G, K, V><<<grid, THREADS_OF<G>, smem, rt().stream>>>(p);
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
        const size_t smem = ROWS_OF<G> * std::max(Ahead<G, K, V, 2>::FLOATS, (size_t)2 * C) * sizeof(float);
        int grid;
        static PerSm known;
        if (int s = resident_grid(known, (const void *)norm_bwd_kernel<G, K, V>, THREADS_OF<G>, smem, rows, ROWS_OF<G>, &grid)) return s;
        float *partial = (float *)scratch_alloc((size_t)grid * 2 * C * sizeof(float));
        if (!partial) return (int)SEERA_E_OOM;
        const NormBwd p{dy, x, gamma, stats, dx, partial, rows, C, kind};
        norm_bwd_kernel<G, K, V><<<grid, THREADS_OF<G>, smem, rt().stream>>>(p);
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
        const int grid = (int)(((long long)rows + ROWS_OF<G> - 1) / ROWS_OF<G>);
        residual_fwd_kernel<G, K, V><<<grid, THREADS_OF<G>, 0, rt().stream>>>(p);
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
        const size_t smem = ROWS_OF<G> * std::max(Ahead<G, K, V, 5>::FLOATS, (size_t)sums * C) * sizeof(float);
        int grid;
        static PerSm known;
        if (int s = resident_grid(known, (const void *)residual_bwd_kernel<G, K, V>, THREADS_OF<G>, smem, rows, ROWS_OF<G>, &grid)) return s;
        float *partial = (float *)scratch_alloc((size_t)grid * sums * C * sizeof(float));
        if (!partial) return (int)SEERA_E_OOM;
        const ResidualBwd p{dout, dy, u, gate, res, gamma, scale, next_gamma, stats, du, dgate, dres, partial, ld_gate, ld_dgate, rows, C, kind, act, next_kind};
        residual_bwd_kernel<G, K, V><<<grid, THREADS_OF<G>, smem, rt().stream>>>(p);
        count_launch();
        int s = check_cuda(cudaGetLastError(), "gated_residual_bwd");
        if (!s) s = param_sums(partial, {{dgamma, dscale, dnext_gamma, dnext_beta}}, C, sums, grid, "gated_residual_bwd(sums)");
        scratch_free(partial);
        return s;
    });
}

}  // extern "C"
