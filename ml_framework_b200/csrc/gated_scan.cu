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
// a = sigmoid(f) and 1 - a, both to full relative precision: a state that decays by 1e-4 a step is summed over ten thousand of them
__device__ __forceinline__ void gates(float f, float &a, float &na) {
    const float e = expf(-fabsf(f)), r = 1.f / (1.f + e), s = e * r;
    a = f >= 0.f ? r : s;
    na = f >= 0.f ? s : r;
    if (f != f) a = na = f;
}

struct ScanFwd {
    const float *f, *v, *h0;
    const int *lengths;
    float *h, *last;
    long long ld;
    int N, T, C;
};
struct ScanBwd {
    const float *f, *v, *h0;
    const int *lengths;
    const float *h, *dh, *dlast;
    float *df, *dv, *dh0;
    long long ld, ldg;
    int N, T, C;
};

__global__ void __launch_bounds__(128) scan_fwd_serial_kernel(const __grid_constant__ ScanFwd p) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= (long long)p.N * p.C) return;
    const int n = (int)(i / p.C), c = (int)(i % p.C);
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.T) : p.T;
    float s = p.h0 ? p.h0[i] : 0.f;
    for (int t = 0; t < p.T; t++) {
        const long long row = (long long)n * p.T + t;
        float o = 0.f;
        if (t < len) {
            float a, na;
            gates(p.f[row * p.ld + c], a, na);
            s = a * s + na * p.v[row * p.ld + c];
            o = s;
        }
        if (p.h) p.h[row * p.C + c] = o;
    }
    if (p.last) p.last[i] = s;
}

__global__ void __launch_bounds__(128) scan_bwd_serial_kernel(const __grid_constant__ ScanBwd p) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= (long long)p.N * p.C) return;
    const int n = (int)(i / p.C), c = (int)(i % p.C);
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.T) : p.T;
    float s = p.dlast ? p.dlast[i] : 0.f;
    for (int t = p.T - 1; t >= 0; t--) {
        const long long row = (long long)n * p.T + t;
        float df = 0.f, dv = 0.f;
        if (t < len) {
            float a, na;
            gates(p.f[row * p.ld + c], a, na);
            const float g = (p.dh ? p.dh[row * p.C + c] : 0.f) + s;
            const float before = t ? p.h[(row - 1) * p.C + c] : (p.h0 ? p.h0[i] : 0.f);
            df = a * na * (before - p.v[row * p.ld + c]) * g;
            dv = na * g;
            s = a * g;
        }
        p.df[row * p.ldg + c] = df;
        p.dv[row * p.ldg + c] = dv;
    }
    if (p.dh0) p.dh0[i] = s;
}
}  // namespace

}  // namespace seera

using namespace seera;

extern "C" {

int seera_gated_scan_fwd(const float *gate, const float *cand, int ld, const float *h0, const int *lengths, float *h, float *h_last, int N, int T,
                         int C) {
    SEERA_ENSURE();
    if (N < 0 || T < 0 || C < 1 || ld < C || (!h && !h_last) || (N > 0 && T > 0 && (!gate || !cand))) return fail(SEERA_E_ARG, "gated_scan_fwd: bad argument");
    if ((long long)N * C > 0x7fffffffLL) return fail(SEERA_E_LIMIT, "gated_scan_fwd: %lld states", (long long)N * C);
    if (N == 0) return SEERA_OK;
    const ScanFwd p{gate, cand, h0, lengths, h, h_last, ld, N, T, C};
    ProfBytes pb((8.0 + (h ? 4 : 0)) * N * T * C, "gated_scan_fwd");
    scan_fwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
    SEERA_LAUNCH_CHECK("gated_scan_fwd");
    return SEERA_OK;
}

int seera_gated_scan_bwd(const float *gate, const float *cand, int ld, const float *h0, const int *lengths, const float *h, const float *dh,
                         const float *dh_last, float *dgate, float *dcand, int ld_grad, float *dh0, int N, int T, int C) {
    SEERA_ENSURE();
    if (N < 0 || T < 0 || C < 1 || ld < C || ld_grad < C || (N > 0 && T > 0 && (!gate || !cand || !h || !dgate || !dcand)) || (!dh && !dh_last))
        return fail(SEERA_E_ARG, "gated_scan_bwd: bad argument");
    if ((long long)N * C > 0x7fffffffLL) return fail(SEERA_E_LIMIT, "gated_scan_bwd: %lld states", (long long)N * C);
    if (N == 0) return SEERA_OK;
    const ScanBwd p{gate, cand, h0, lengths, h, dh, dh_last, dgate, dcand, dh0, ld, ld_grad, N, T, C};
    ProfBytes pb((20.0 + (dh ? 4 : 0)) * N * T * C, "gated_scan_bwd");
    scan_bwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
    SEERA_LAUNCH_CHECK("gated_scan_bwd");
    return SEERA_OK;
}

}  // extern "C"
