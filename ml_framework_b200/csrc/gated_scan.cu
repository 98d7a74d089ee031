// Gated linear recurrence over the time axis, per sequence and channel, with a = sigmoid(gate):
//
//   h[t] = a[t] h[t-1] + (1 - a[t]) v[t],   h[-1] = h0 (0 without one)
//
// and its gradients from dh and dh_last, going back in time:
//
//   g[t] = dh[t] + c[t+1],  c[t] = a[t] g[t],  c[length] = dh_last
//   dv = (1 - a) g,   dgate = a (1 - a) (h[t-1] - v[t]) g,   dh0 = c[0]
//
// Steps at and behind a sequence's length hold the state, write zeros and are not read.
#include "common.cuh"

namespace seera {

namespace {
struct ScanFwd {
    const float *f, *v, *h0;
    const int *lengths;
    float *h, *last;
    long long ld;
    int N, T, C, ranks;
};
struct ScanBwd {
    const float *f, *v, *h0;
    const int *lengths;
    const float *h, *dh, *dlast;
    float *df, *dv, *dh0;
    long long ld, ldg;
    int N, T, C, ranks;
};

// A gate is kept as the smaller of a and 1 - a, which has its full relative precision, with the sign bit where that is a: a state that decays by
// 1e-4 a step is summed over ten thousand of them, and one minus a rounded a would have lost four of seven digits there.
__device__ __forceinline__ float gate_of(float f) {
    const float s = __fdividef(1.f, 1.f + expf(fabsf(f)));
    return f > 0.f ? s : -s;
}
constexpr float HOLD = 0.f;                               // the gate of a step that is not there: a = 1
__device__ __forceinline__ bool keeps(float s) { return __float_as_int(s) >= 0; }       // (the sign of a zero counts)
// a h + (1 - a) v
__device__ __forceinline__ float step_of(float s, float h, float v) {
    const bool k = keeps(s);
    const float base = k ? h : v, to = k ? v : h;
    return fmaf(fabsf(s), to - base, base);
}
// a x, and with (1 - a) x beside it
__device__ __forceinline__ float decay(float s, float x) {
    const float y = fabsf(s) * x;
    return keeps(s) ? x - y : y;
}
__device__ __forceinline__ void part(float s, float x, float &a_x, float &na_x) {
    const float y = fabsf(s) * x, z = x - y;
    a_x = keeps(s) ? z : y;
    na_x = keeps(s) ? y : z;
}

__device__ __forceinline__ int length_of(const int *lengths, int n, int T) { return lengths ? min(max(lengths[n], 0), T) : T; }

// A thread per state, step by step; AHEAD steps are requested before the first of them is worked on.
constexpr int AHEAD = 4;
__global__ void __launch_bounds__(128) scan_fwd_serial_kernel(const __grid_constant__ ScanFwd p) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= (long long)p.N * p.C) return;
    const int n = (int)(i / p.C), c = (int)(i - (long long)n * p.C), len = length_of(p.lengths, n, p.T);
    const float *f = p.f + (long long)n * p.T * p.ld + c, *v = p.v + (long long)n * p.T * p.ld + c;
    float *h = p.h ? p.h + (long long)n * p.T * p.C + c : nullptr;
    float s = p.h0 ? p.h0[i] : 0.f;
    for (int t = 0; t < p.T; t += AHEAD) {
        float ff[AHEAD], vv[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (t + k < len) { ff[k] = f[(t + k) * p.ld]; vv[k] = v[(t + k) * p.ld]; }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (t + k >= p.T) break;
            if (t + k < len) s = step_of(gate_of(ff[k]), s, vv[k]);
            if (h) h[(long long)(t + k) * p.C] = t + k < len ? s : 0.f;
        }
    }
    if (p.last) p.last[i] = s;
}

__global__ void __launch_bounds__(128) scan_bwd_serial_kernel(const __grid_constant__ ScanBwd p) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= (long long)p.N * p.C) return;
    const int n = (int)(i / p.C), c = (int)(i - (long long)n * p.C), len = length_of(p.lengths, n, p.T);
    const long long at = (long long)n * p.T;
    float s = p.dlast ? p.dlast[i] : 0.f;
    for (int t = p.T - 1; t >= 0; t--) {
        const long long row = at + t;
        float df = 0.f, dv = 0.f;
        if (t < len) {
            const float gate = gate_of(p.f[row * p.ld + c]), g = (p.dh ? p.dh[row * p.C + c] : 0.f) + s;
            const float before = t ? p.h[(row - 1) * p.C + c] : (p.h0 ? p.h0[i] : 0.f);
            part(gate, g, s, dv);
            df = (1.f - fabsf(gate)) * (fabsf(gate) * g) * (before - p.v[row * p.ld + c]);
        }
        p.df[row * p.ldg + c] = df;
        p.dv[row * p.ldg + c] = dv;
    }
    if (p.dh0) p.dh0[i] = s;
}

// ---- time split over warps and over the blocks of a cluster ---------------------------------------------------------------------------
// A lane has one channel (a warp reads whole lines), a warp STEPS neighbouring steps of it in registers, a block WARPS of those and the blocks of a
// cluster follow one another; the cluster then goes on to the next such piece of time, whose loads are on their way meanwhile.  What a run of steps
// does to a state is one multiply-add, x -> A x + B: warps put theirs into shared memory, blocks send theirs to the others of the cluster, and
// with the state at its start every warp goes over its registers again and writes.  One barrier of the block and one of the cluster a piece, with the
// places in shared memory used in turn.
constexpr int WARPS = 8, FWD_STEPS = 16, BWD_STEPS = 8, MAX_RANKS = 8;

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void send(float2 *mine, int rank, float2 v) {
    unsigned local = (unsigned)__cvta_generic_to_shared(mine), remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ float2 then(float2 first, float2 second) { return make_float2(first.x * second.x, fmaf(second.x, first.y, second.y)); }

struct Joined {
    float2 warps[2][WARPS][32], ranks[2][MAX_RANKS][32];
};
// The state at the start of this warp's steps, from that at the start of the piece; `carry` goes on to the start of the next one.
__device__ __forceinline__ float join(Joined &sm, int buf, float2 mine, int warp, int lane, int rank, int ranks, float &carry) {
    sm.warps[buf][warp][lane] = mine;
    __syncthreads();
    float2 before = make_float2(1.f, 0.f), all = before;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        if (w == warp) before = all;
        all = then(all, sm.warps[buf][w][lane]);
    }
    float x = carry;
    if (ranks > 1) {
        if (warp < ranks) send(&sm.ranks[buf][rank][lane], warp, all);        // a warp for each block of the cluster (at most WARPS of them)
        cluster_sync();
        for (int r = 0; r < ranks; r++) {
            if (r == rank) x = carry;
            const float2 o = sm.ranks[buf][r][lane];
            carry = fmaf(o.x, carry, o.y);
        }
    } else {
        carry = fmaf(all.x, carry, all.y);
    }
    return fmaf(before.x, x, before.y);
}

__global__ void __launch_bounds__(WARPS * 32, 2) scan_fwd_kernel(const __grid_constant__ ScanFwd p) {
    constexpr int L = FWD_STEPS;
    __shared__ Joined sm;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x % p.ranks, tiles = (p.C + 31) / 32;
    const unsigned tile = blockIdx.x / p.ranks;
    const int n = tile / tiles, c = (tile - n * tiles) * 32 + lane;
    const bool on = c < p.C;
    const int len = on ? length_of(p.lengths, n, p.T) : 0;
    const long long at = (long long)n * p.T;
    const int piece = p.ranks * WARPS * L;
    float carry = on && p.h0 ? p.h0[(long long)n * p.C + c] : 0.f;
    float f[L], v[L];
    auto request = [&](int t0) {
        const float *pf = p.f + (at + t0) * p.ld + c, *pv = p.v + (at + t0) * p.ld + c;
#pragma unroll
        for (int i = 0; i < L; i++)
            if (t0 + i < len) { f[i] = __ldcs(pf + i * p.ld); v[i] = __ldcs(pv + i * p.ld); }
    };
    int t0 = (rank * WARPS + warp) * L, buf = 0;
    request(t0);
    if (p.ranks > 1) cluster_sync();                        // the others' shared memory is there
    for (int start = 0; start < p.T; start += piece, t0 += piece, buf ^= 1) {
        float s[L], u[L];
        float2 mine = make_float2(1.f, 0.f);
#pragma unroll
        for (int i = 0; i < L; i++) {
            s[i] = HOLD; u[i] = 0.f;
            if (t0 + i < len) { s[i] = gate_of(f[i]); u[i] = v[i]; }
            mine.y = step_of(s[i], mine.y, u[i]);
            mine.x = decay(s[i], mine.x);
        }
        request(t0 + piece);
        float x = join(sm, buf, mine, warp, lane, rank, p.ranks, carry);
        if (p.h && on) {
            float *h = p.h + (at + t0) * p.C + c;
#pragma unroll
            for (int i = 0; i < L; i++) {
                x = step_of(s[i], x, u[i]);
                if (t0 + i < p.T) __stcs(h + (long long)i * p.C, t0 + i < len ? x : 0.f);
            }
        }
    }
    if (on && p.last && rank == 0 && warp == 0) p.last[(long long)n * p.C + c] = carry;
}

// Backward: the same with time running from the end, where c -> a (dh + c) is what a step does.
__global__ void __launch_bounds__(WARPS * 32, 2) scan_bwd_kernel(const __grid_constant__ ScanBwd p) {
    constexpr int L = BWD_STEPS;
    __shared__ Joined sm;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x % p.ranks, tiles = (p.C + 31) / 32;
    const unsigned tile = blockIdx.x / p.ranks;
    const int n = tile / tiles, c = (tile - n * tiles) * 32 + lane;
    const bool on = c < p.C;
    const int len = on ? length_of(p.lengths, n, p.T) : 0;
    const long long at = (long long)n * p.T, state = (long long)n * p.C + c;
    const int piece = p.ranks * WARPS * L;
    float carry = on && p.dlast ? p.dlast[state] : 0.f;
    float f[L], v[L], d[L], b[L];
    auto request = [&](int t1) {                            // steps t1, t1 - 1, ...
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int t = t1 - i;
            if (t >= 0 && t < len) {
                const long long row = at + t;
                f[i] = __ldcs(p.f + row * p.ld + c);
                v[i] = __ldcs(p.v + row * p.ld + c);
                d[i] = p.dh ? __ldcs(p.dh + row * p.C + c) : 0.f;
                b[i] = t ? __ldcs(p.h + (row - 1) * p.C + c) : (p.h0 ? p.h0[state] : 0.f);
            }
        }
    };
    int t1 = p.T - 1 - (rank * WARPS + warp) * L, buf = 0;
    request(t1);
    if (p.ranks > 1) cluster_sync();
    for (int start = 0; start < p.T; start += piece, t1 -= piece, buf ^= 1) {
        float s[L], e[L], w[L];
        float2 mine = make_float2(1.f, 0.f);
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int t = t1 - i;
            s[i] = HOLD; e[i] = 0.f; w[i] = 0.f;
            if (t >= 0 && t < len) { s[i] = gate_of(f[i]); e[i] = d[i]; w[i] = b[i] - v[i]; }
            mine.y = decay(s[i], e[i] + mine.y);
            mine.x = decay(s[i], mine.x);
        }
        request(t1 - piece);
        float x = join(sm, buf, mine, warp, lane, rank, p.ranks, carry);
        if (on) {
#pragma unroll
            for (int i = 0; i < L; i++) {
                const int t = t1 - i;
                if (t < 0) break;
                const float g = e[i] + x, small = fabsf(s[i]);
                float dv;
                part(s[i], g, x, dv);
                const bool there = t < len;
                __stcs(p.df + (at + t) * p.ldg + c, there ? (1.f - small) * (small * g) * w[i] : 0.f);
                __stcs(p.dv + (at + t) * p.ldg + c, there ? dv : 0.f);
            }
        }
    }
    if (on && p.dh0 && rank == 0 && warp == 0) p.dh0[state] = carry;
}

// Blocks of a cluster: as many as it takes to give every SM two blocks, and no more than there are steps for.
int ranks_of(int N, int T, int C, int steps) {
    const long long tiles = (long long)N * ((C + 31) / 32);
    int k = 1;
    while (k < MAX_RANKS && tiles * k < 2 * rt().sm_count && (long long)k * WARPS * steps < T) k *= 2;
    return k;
}
template <class P> cudaError_t launch_clusters(void (*kernel)(P), const P &p, long long tiles) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.ranks)); cfg.blockDim = dim3(WARPS * 32); cfg.stream = rt().stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = p.ranks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}
// Few steps: a thread per state has nothing to split.
constexpr int SERIAL_STEPS = 16;
}  // namespace

}  // namespace seera

using namespace seera;

extern "C" {

int seera_gated_scan_fwd(const float *gate, const float *cand, int ld, const float *h0, const int *lengths, float *h, float *h_last, int N, int T,
                         int C) {
    SEERA_ENSURE();
    if (N < 0 || T < 0 || C < 1 || ld < C || (!h && !h_last) || (N > 0 && T > 0 && (!gate || !cand))) return fail(SEERA_E_ARG, "gated_scan_fwd: bad argument");
    if ((long long)N * C > 0x7fffffffLL || T > (1 << 30)) return fail(SEERA_E_LIMIT, "gated_scan_fwd: %lld states, %d steps", (long long)N * C, T);
    if (N == 0) return SEERA_OK;
    const ScanFwd p{gate, cand, h0, lengths, h, h_last, ld, N, T, C, ranks_of(N, T, C, FWD_STEPS)};
    ProfBytes pb((8.0 + (h ? 4 : 0)) * N * T * C, "gated_scan_fwd");
    if (T <= SERIAL_STEPS) scan_fwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
    else launch_clusters(scan_fwd_kernel, p, (long long)N * ((C + 31) / 32));
    SEERA_LAUNCH_CHECK("gated_scan_fwd");
    return SEERA_OK;
}

int seera_gated_scan_bwd(const float *gate, const float *cand, int ld, const float *h0, const int *lengths, const float *h, const float *dh,
                         const float *dh_last, float *dgate, float *dcand, int ld_grad, float *dh0, int N, int T, int C) {
    SEERA_ENSURE();
    if (N < 0 || T < 0 || C < 1 || ld < C || ld_grad < C || (N > 0 && T > 0 && (!gate || !cand || !h || !dgate || !dcand)) || (!dh && !dh_last))
        return fail(SEERA_E_ARG, "gated_scan_bwd: bad argument");
    if ((long long)N * C > 0x7fffffffLL || T > (1 << 30)) return fail(SEERA_E_LIMIT, "gated_scan_bwd: %lld states, %d steps", (long long)N * C, T);
    if (N == 0) return SEERA_OK;
    const ScanBwd p{gate, cand, h0, lengths, h, dh, dh_last, dgate, dcand, dh0, ld, ld_grad, N, T, C, ranks_of(N, T, C, BWD_STEPS)};
    ProfBytes pb((20.0 + (dh ? 4 : 0)) * N * T * C, "gated_scan_bwd");
    if (T <= SERIAL_STEPS) scan_bwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
    else launch_clusters(scan_bwd_kernel, p, (long long)N * ((C + 31) / 32));
    SEERA_LAUNCH_CHECK("gated_scan_bwd");
    return SEERA_OK;
}

}  // extern "C"
