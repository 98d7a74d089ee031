// One AdamW step over many tensors, with its averages in 32 bits or in 8.
//
//   g = grad_scale * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  w = (1 - lr decay) w - lr (m / c1) / (sqrt(v / c2) + eps)
//
// The tensors of a step travel as a table in the kernel's arguments: nothing is uploaded, a recorded launch carries its own copy, and a
// step of a small network is one launch.  A block takes CHUNK neighbouring entries of one tensor, which it finds by bisection in the table.
// A chunk belongs to one tensor, so that a tensor's decay is the block's.
//
// What bounds it: the bytes.  32 bits: w, m, v read and written and the gradient read, 28 bytes an entry.  8 bits: 12 for w and the gradient
// and 2 x 136 / 64 for the averages.
//
// Averages in 8 bits.  64 neighbouring entries of a tensor share a block of 136 bytes: sixteen times four codes of m and four of v (what a
// thread reads and writes, in one piece), then the largest |m| and the largest v as floats.  A code is an entry over the block's largest, as a
// small float: m a sign, 4 bits of exponent and 3 of mantissa (down to 2^-17 of the largest), v 5 bits of exponent and 3 of mantissa (down to
// 2^-33: v is a square).  The bits of a float times 2^-112 (2^-96) hold that code in their places 20 and up, the float's own denormals
// serving as the code's, so both ways are one multiplication and one shift.
// Rounding goes up with the probability of the distance gone, from 16 random bits each: the code's mean is the value.  Rounded to nearest, v would
// stand still: beta2 = 0.999 moves it by at most 0.1 % of itself a step where half a code is 3 to 6 %.  The random bits are a hash of the
// entry's place and the step, so a step is reproducible.  The weights are updated from the averages as they are before rounding.
#include "common.cuh"
#include "internal.h"
#include <memory>
#include <string.h>

namespace seera {

namespace {
constexpr int CHUNK = 2048, THREADS = 256;
constexpr int TABLE = 80;                     // tensors of one launch: with the scalars just under 4 KB of arguments

struct AdamWTensor {
    float *w;
    const float *g;
    void *m;                                  // 8 bits: the blocks of both averages
    union { float *v; long long place; };     // 8 bits: number of the tensor's first entry, for the random bits
    long long n;
    float decay;
    unsigned first;                           // first block of the launch that works on it
};
struct AdamWTable {
    AdamWTensor t[TABLE];
    const float *hyper;                       // where not null, the scalars are there
    int count;
};
struct AdamWArgs { float lr, b1, omb1, b2, omb2, eps, c1, c2, gs, step; };
static_assert(sizeof(AdamWTable) + sizeof(AdamWArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ AdamWArgs adamw_args(const AdamWTable &tab, const AdamWArgs &by_value, bool eight) {
    if (!tab.hyper) return by_value;
    const float *h = tab.hyper;
    return AdamWArgs{h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[7], h[8], eight ? h[9] : 0.f};
}
__device__ __forceinline__ int tensor_of(const AdamWTable &tab, unsigned block) {
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.t[mid].first <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// What a step needs of the scalars: w = keep w - rate m / (root sqrt(v) + eps).
struct Update { float keep, rate, root; };
__device__ __forceinline__ Update update_of(const AdamWArgs &a, float decay) { return Update{1.f - a.lr * decay, a.lr / a.c1, 1.f / sqrtf(a.c2)}; }
// Every operation on the averages rounded by itself: the codes of the 8-bit form follow from these bits, and both forms keep the same averages.  The
// weight's step takes the approximate square root (2^-23) and division (2^-22): of the step, which is a small part of the weight.
__device__ __forceinline__ void adamw_one(float &w, float g, float &m, float &v, const AdamWArgs &a, const Update &u) {
    g = __fmul_rn(g, a.gs);
    m = __fadd_rn(__fmul_rn(a.b1, m), __fmul_rn(a.omb1, g));
    v = __fadd_rn(__fmul_rn(a.b2, v), __fmul_rn(a.omb2, __fmul_rn(g, g)));
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    w = fmaf(w, u.keep, -__fdividef(u.rate * m, fmaf(r, u.root, a.eps)));
}

__global__ void __launch_bounds__(THREADS) adamw_kernel(const __grid_constant__ AdamWTable tab, const __grid_constant__ AdamWArgs by_value) {
    const AdamWTensor &t = tab.t[tensor_of(tab, blockIdx.x)];
    const AdamWArgs a = adamw_args(tab, by_value, false);
    const Update u = update_of(a, t.decay);
    const long long at = (long long)(blockIdx.x - t.first) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.n - at);
    float *w = t.w + at, *m = (float *)t.m + at, *v = t.v + at;
    const float *g = t.g + at;
    if (n == CHUNK && !(((uintptr_t)w | (uintptr_t)m | (uintptr_t)v | (uintptr_t)g) & 15)) {
        float4 ww[2], gg[2], mm[2], vv[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = threadIdx.x + k * THREADS;
            ww[k] = ((float4 *)w)[i]; gg[k] = __ldcs((const float4 *)g + i); mm[k] = ((float4 *)m)[i]; vv[k] = ((float4 *)v)[i];
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = threadIdx.x + k * THREADS;
            adamw_one(ww[k].x, gg[k].x, mm[k].x, vv[k].x, a, u); adamw_one(ww[k].y, gg[k].y, mm[k].y, vv[k].y, a, u);
            adamw_one(ww[k].z, gg[k].z, mm[k].z, vv[k].z, a, u); adamw_one(ww[k].w, gg[k].w, mm[k].w, vv[k].w, a, u);
            ((float4 *)w)[i] = ww[k]; ((float4 *)m)[i] = mm[k]; ((float4 *)v)[i] = vv[k];
        }
        return;
    }
    for (int i = threadIdx.x; i < n; i += THREADS) {
        float ww = w[i], mm = m[i], vv = v[i];
        adamw_one(ww, g[i], mm, vv, a, u);
        w[i] = ww; m[i] = mm; v[i] = vv;
    }
}

constexpr int BLOCK_ENTRIES = 64, BLOCK_BYTES = 136;
constexpr float M_UNIT = 0x1p-112f, V_UNIT = 0x1p-96f;       // 1.0 times these has the exponent fields 15 and 31: the largest codes
constexpr unsigned M_TOP = 0x78, V_TOP = 0xF8;

// The hash of a place and a step, its first line apart: four neighbouring places from a multiple of four on differ in it by their last two bits.
__device__ __forceinline__ unsigned random_seed(unsigned long long place, unsigned step) {
    return (unsigned)place ^ ((unsigned)(place >> 32) * 0x632BE5ABu) ^ (step * 0x9E3779B1u);
}
__device__ __forceinline__ unsigned random32(unsigned x) {
    x = (x ^ (x >> 16)) * 0xA3D95F4Bu;
    x = (x ^ (x >> 15)) * 0x6C8E9D73u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ float decode_m(unsigned c, float largest) {
    const float x = __fmul_rn(__fmul_rn(__uint_as_float((c & 127u) << 20), 1.f / M_UNIT), largest);
    return c & 128u ? -x : x;
}
__device__ __forceinline__ float decode_v(unsigned c, float largest) { return __fmul_rn(__fmul_rn(__uint_as_float(c << 20), 1.f / V_UNIT), largest); }
__device__ __forceinline__ unsigned encode(float x, float inv, float unit, unsigned top, unsigned random16) {
    return min((__float_as_uint(__fmul_rn(__fmul_rn(x, inv), unit)) + (random16 << 4)) >> 20, top);
}
// A block whose largest entry is below the smallest normal float is held as zeros.
__device__ __forceinline__ float largest_of(unsigned bits, float &inv) {
    float x = __uint_as_float(bits);
    if (x < 1.17549435e-38f) x = 0.f;
    inv = x > 0.f ? __frcp_rn(x) : 0.f;
    return x;
}

__global__ void __launch_bounds__(THREADS) adamw8_kernel(const __grid_constant__ AdamWTable tab, const __grid_constant__ AdamWArgs by_value) {
    const AdamWTensor &t = tab.t[tensor_of(tab, blockIdx.x)];
    const AdamWArgs a = adamw_args(tab, by_value, true);
    const Update u = update_of(a, t.decay);
    const unsigned step = (unsigned)a.step;
    const long long at = (long long)(blockIdx.x - t.first) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.n - at);
    float *w = t.w + at;
    const float *g = t.g + at;
    char *state = (char *)t.m + at / BLOCK_ENTRIES * BLOCK_BYTES;
    const bool vec = !(((uintptr_t)w | (uintptr_t)g) & 15);
    const int part = threadIdx.x & 15;                        // 16 threads a block of 64 entries
    float ww[2][4], gg[2][4];
    uint2 code[2];
    float2 top[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = (threadIdx.x + k * THREADS) * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) ww[k][j] = gg[k][j] = 0.f;
        code[k] = make_uint2(0, 0);
        top[k] = make_float2(0.f, 0.f);
        if (i / BLOCK_ENTRIES * BLOCK_ENTRIES < n) {          // the tensor's last block may be short, its codes are there for all 64
            const char *blk = state + i / BLOCK_ENTRIES * BLOCK_BYTES;
            code[k] = ((const uint2 *)blk)[part];
            top[k] = *(const float2 *)(blk + 128);
        }
        if (vec && i + 4 <= n) {
            const float4 x = *(const float4 *)(w + i), y = __ldcs((const float4 *)(g + i));
            ww[k][0] = x.x; ww[k][1] = x.y; ww[k][2] = x.z; ww[k][3] = x.w;
            gg[k][0] = y.x; gg[k][1] = y.y; gg[k][2] = y.z; gg[k][3] = y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) if (i + j < n) { ww[k][j] = w[i + j]; gg[k][j] = g[i + j]; }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = (threadIdx.x + k * THREADS) * 4;
        float m[4], v[4];
        unsigned am = 0, av = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            m[j] = decode_m((code[k].x >> (8 * j)) & 255u, top[k].x);
            v[j] = decode_v((code[k].y >> (8 * j)) & 255u, top[k].y);
            adamw_one(ww[k][j], gg[k][j], m[j], v[j], a, u);
            if (i + j >= n) m[j] = v[j] = 0.f;                // places behind the tensor's end
            am = max(am, __float_as_uint(m[j]) & 0x7fffffffu);      // as bits: a NaN is larger than all else, and its block shows it
            av = max(av, __float_as_uint(v[j]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) {
            am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
            av = max(av, __shfl_xor_sync(0xffffffffu, av, o));
        }
        float im, iv;
        const float lm = largest_of(am, im), lv = largest_of(av, iv);
        uint2 c = make_uint2(0, 0);
        const unsigned seed = random_seed((unsigned long long)(t.place + at + i), step);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned r = random32(seed ^ j);
            c.x |= (encode(fabsf(m[j]), im, M_UNIT, M_TOP, r & 0xffffu) | (m[j] < 0.f ? 128u : 0u)) << (8 * j);
            c.y |= encode(v[j], iv, V_UNIT, V_TOP, r >> 16) << (8 * j);
        }
        if (i / BLOCK_ENTRIES * BLOCK_ENTRIES < n) {
            char *blk = state + i / BLOCK_ENTRIES * BLOCK_BYTES;
            ((uint2 *)blk)[part] = c;
            if (part == 0) *(float2 *)(blk + 128) = make_float2(lm, lv);
        }
        if (vec && i + 4 <= n) *(float4 *)(w + i) = make_float4(ww[k][0], ww[k][1], ww[k][2], ww[k][3]);
        else {
#pragma unroll
            for (int j = 0; j < 4; j++) if (i + j < n) w[i + j] = ww[k][j];
        }
    }
}

__global__ void __launch_bounds__(256) adamw8_read_kernel(const char *__restrict__ state, float *__restrict__ m, float *__restrict__ v, long long n) {
    const bool vec = !(((uintptr_t)m | (uintptr_t)v) & 15);
    for (long long p = (long long)blockIdx.x * 256 + threadIdx.x; p * 4 < n; p += (long long)gridDim.x * 256) {
        const char *blk = state + p / 16 * BLOCK_BYTES;
        const uint2 c = ((const uint2 *)blk)[p & 15];
        const float2 top = *(const float2 *)(blk + 128);
        float x[4], y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) { x[j] = decode_m((c.x >> (8 * j)) & 255u, top.x); y[j] = decode_v((c.y >> (8 * j)) & 255u, top.y); }
        const long long i = p * 4;
        if (vec && i + 4 <= n) {
            *(float4 *)(m + i) = make_float4(x[0], x[1], x[2], x[3]);
            *(float4 *)(v + i) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) if (i + j < n) { m[i + j] = x[j]; v[i + j] = y[j]; }
        }
    }
}

int adamw(bool eight, int count, float *const *w, const float *const *g, void *const *m, float *const *v, const long long *n, const float *decay,
          const AdamWArgs &a, const float *hyper, long long first, const char *name) {
    SEERA_ENSURE();
    if (count < 0 || (count > 0 && (!w || !g || !m || !n || !decay || (!eight && !v))) || first < 0 || first % BLOCK_ENTRIES) return fail(SEERA_E_ARG, "%s: bad argument", name);
    double total = 0;
    for (int i = 0; i < count; i++) {
        if (n[i] < 0 || (n[i] > 0 && (!w[i] || !g[i] || !m[i] || (!eight && !v[i])))) return fail(SEERA_E_ARG, "%s: bad argument for tensor %d", name, i);
        if (n[i] > (1LL << 40)) return fail(SEERA_E_LIMIT, "%s: tensor %d has %lld entries", name, i, n[i]);
        if (eight && ((uintptr_t)m[i] & 7)) return fail(SEERA_E_ARG, "%s: the state of tensor %d does not start on 8 bytes", name, i);
        total += (double)n[i];
    }
    if (total == 0) return SEERA_OK;
    ProfBytes pb((eight ? 12.0 + 2.0 * BLOCK_BYTES / BLOCK_ENTRIES : 28.0) * total, name);
    const void *kernel = eight ? (const void *)adamw8_kernel : (const void *)adamw_kernel;
    auto table = std::make_shared<AdamWTable>();
    AdamWArgs args = a;
    for (int i = 0; i < count;) {
        memset(table.get(), 0, sizeof(AdamWTable));
        table->hyper = hyper;
        long long blocks = 0;
        for (; i < count && table->count < TABLE; i++) {
            if (n[i] == 0) continue;
            const long long need = (n[i] + CHUNK - 1) / CHUNK;
            if (blocks + need > 0x7fffffffLL) break;
            AdamWTensor &t = table->t[table->count++];
            t.w = w[i]; t.g = g[i]; t.m = m[i]; t.n = n[i]; t.decay = decay[i]; t.first = (unsigned)blocks;
            if (eight) t.place = first;
            else t.v = v[i];
            blocks += need;
            if (eight) first += (n[i] + BLOCK_ENTRIES - 1) / BLOCK_ENTRIES * BLOCK_ENTRIES;
        }
        if (!table->count) break;                             // tensors without entries were the last
        void *argv[] = {table.get(), &args};
        cudaLaunchKernel(kernel, dim3((unsigned)blocks), dim3(THREADS), argv, 0, rt().stream);
        SEERA_LAUNCH_CHECK(name);
        if (rt().capturing && !hyper) {
            OptLaunch l = {};
            l.kind = 2; l.grid = (int)blocks; l.n_scalars = eight ? 10 : 9;
            memcpy(l.scalars, &args, sizeof(float) * l.n_scalars);
            l.func = kernel;
            l.table = table;
            if (int s = graph_note_optimizer(l)) return s;
            table = std::make_shared<AdamWTable>();
        }
    }
    return SEERA_OK;
}
}  // namespace

}  // namespace seera

using namespace seera;

extern "C" {

int seera_adamw_step(int count, float *const *w, const float *const *g, float *const *m, float *const *v, const long long *n, const float *decay,
                     float lr, float beta1, float omb1, float beta2, float omb2, float eps, float c1, float c2, float grad_scale,
                     const float *hyper) {
    return adamw(false, count, w, g, (void *const *)m, v, n, decay, {lr, beta1, omb1, beta2, omb2, eps, c1, c2, grad_scale, 0.f}, hyper, 0,
                 "adamw_step");
}

size_t seera_adamw8_state_bytes(long long n) { return n < 0 ? 0 : (size_t)((n + BLOCK_ENTRIES - 1) / BLOCK_ENTRIES) * BLOCK_BYTES; }

int seera_adamw8_step(int count, float *const *w, const float *const *g, void *const *state, const long long *n, const float *decay, float lr,
                      float beta1, float omb1, float beta2, float omb2, float eps, float c1, float c2, float grad_scale, float step,
                      const float *hyper, long long first) {
    if (!(step >= 0.f && step < 4294967040.f) && !hyper) return fail(SEERA_E_ARG, "adamw8_step: step %g", (double)step);
    return adamw(true, count, w, g, state, nullptr, n, decay, {lr, beta1, omb1, beta2, omb2, eps, c1, c2, grad_scale, step}, hyper, first,
                 "adamw8_step");
}

int seera_adamw8_read(const void *state, float *m, float *v, long long n) {
    SEERA_ENSURE();
    if (n < 0 || (n > 0 && (!state || !m || !v)) || ((uintptr_t)state & 7)) return fail(SEERA_E_ARG, "adamw8_read: bad argument");
    if (n == 0) return SEERA_OK;
    adamw8_read_kernel<<<stride_grid((n + 3) / 4), 256, 0, rt().stream>>>((const char *)state, m, v, n);
    SEERA_LAUNCH_CHECK("adamw8_read");
    return SEERA_OK;
}

}  // extern "C"
