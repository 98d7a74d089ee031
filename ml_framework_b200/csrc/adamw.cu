// One AdamW step over many tensors, with its averages in 32 bits or in 8.
//
//   g = grad_scale * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  w = (1 - lr decay) w - lr (m / c1) / (sqrt(v / c2) + eps)
//
// The tensors of a step travel as a table in the kernel's arguments: nothing is uploaded, a recorded launch carries its own copy, and a
// step of a small network is one launch.  A block takes CHUNK neighbouring entries of one tensor, which it finds by bisection in the table.
// A chunk belongs to one tensor, so that a tensor's decay is the block's.
//
// What bounds it: the bytes.  32 bits: w, m, v read and written and the gradient read, 28 bytes an entry; of 67 million entries 277 us, 6.8 TB/s.  8 bits: 12 for w and the gradient
// and 2 x 136 / 64 for the averages; of 67 million entries 180 us, 6.1 TB/s (and 102 us to read them out, 6.7), when an entry takes 40 instructions.
// With four entries a thread, one at a time and with exact roots and divisions it took 107 instructions and 300 us: the instructions bounded it.
//
// Averages in 8 bits.  64 neighbouring entries of a tensor share a block of 136 bytes: sixteen times four codes of m and four of v (what a
// thread reads and writes, in one piece), then the largest |m| and the largest v as floats.  A code is an entry over the block's largest, as a
// small float: m a sign, 4 bits of exponent and 3 of mantissa (down to 2^-17 of the largest), v 5 bits of exponent and 3 of mantissa (down to
// 2^-33: v is a square).  The bits of a float times 2^-112 (2^-96) hold that code in their places 20 and up, the float's own denormals
// serving as the code's, so both ways are one multiplication and one shift.
// Rounding goes up with the probability of the distance gone, from 16 random bits each: the code's mean is the value.  Rounded to nearest, v would
// stand still: beta2 = 0.999 moves it by at most 0.1 % of itself a step where half a code is 3 to 6 %.  The random bits are a hash of the
// entry's place and the step, so a step is reproducible.  The weights are updated from the averages as they are before rounding.
// Bounded steps.  The two averages of an entry are rounded apart: beside an m that went up to 2^-17 of its block's largest a v may go to 0, and the next step divides that m
// by the root of the newest gradient alone.  Entries 2^-17 below their block's largest go up to 1000 lr in a step.  seera_adamw8_bounded_step, which the front
// end's AdamW takes, gives a v above zero the smallest code at least: its root is 2^-16.5, the smallest m is 2^-17.  What lies below both then goes in steps that are too
// small (of 2^-20 a quarter to a half of what 32 bits do), and none is much larger than theirs.  Three instructions an entry: 183 us instead of 180.
#include "common.cuh"
#include "internal.h"
#include "pairs.cuh"
#include <cuda_fp16.h>
#include <memory>
#include <new>
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
};
struct AdamWTable {
    unsigned first[TABLE];                    // of each tensor's blocks; side by side, so that the search waits for few lines of the arguments
    float decay[TABLE];
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
        if (tab.first[mid] <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// What a step needs of the scalars: w = keep w + rate m / (root sqrt(v) + eps).
struct Update { float keep, rate, root; };
__device__ __forceinline__ Update update_of(const AdamWArgs &a, float decay) { return Update{1.f - a.lr * decay, -a.lr / a.c1, 1.f / sqrtf(a.c2)}; }
__device__ __forceinline__ float largest(float a, float b) {            // a NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The approximate square root is off by 2^-23; what lies below the smallest normal number counts as that (the flush would make it zero).
__device__ __forceinline__ float root_of(float v) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(largest(v, 1.17549435e-38f)));
    return r;
}
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// (A sum of two at once would be contracted with the products before it.)
__device__ __forceinline__ Two sum_of(Two a, Two b) { return Two{__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)}; }
// Two entries.  Every operation on the averages rounded by itself: the codes of the 8-bit form follow from these bits, and both forms keep the same
// averages.  The weight's step takes the approximate root and reciprocal (2^-23 each): of the step, which is a small part of the weight.
__device__ __forceinline__ void adamw_two(Two &w, Two g, Two &m, Two &v, const AdamWArgs &a, const Update &u) {
    g = mul2(g, both(a.gs));
    m = sum_of(mul2(both(a.b1), m), mul2(both(a.omb1), g));
    v = sum_of(mul2(both(a.b2), v), mul2(both(a.omb2), mul2(g, g)));
    const Two d = fma2(Two{root_of(v.x), root_of(v.y)}, both(u.root), both(a.eps));
    w = fma2(w, both(u.keep), mul2(mul2(both(u.rate), m), Two{reciprocal(d.x), reciprocal(d.y)}));
}
__device__ __forceinline__ void adamw_one(float &w, float g, float &m, float &v, const AdamWArgs &a, const Update &u) {
    Two ww = both(w), mm = both(m), vv = both(v);
    adamw_two(ww, both(g), mm, vv, a, u);
    w = ww.x; m = mm.x; v = vv.x;
}
struct __align__(16) Four { Two lo, hi; };

__global__ void __launch_bounds__(THREADS) adamw_kernel(const __grid_constant__ AdamWTable tab, const __grid_constant__ AdamWArgs by_value) {
    const int number = tensor_of(tab, blockIdx.x);
    const AdamWTensor &t = tab.t[number];
    const AdamWArgs a = adamw_args(tab, by_value, false);
    const Update u = update_of(a, tab.decay[number]);
    const long long at = (long long)(blockIdx.x - tab.first[number]) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.n - at);
    float *w = t.w + at, *m = (float *)t.m + at, *v = t.v + at;
    const float *g = t.g + at;
    if (n == CHUNK && !(((uintptr_t)w | (uintptr_t)m | (uintptr_t)v | (uintptr_t)g) & 15)) {
        Four ww[2], gg[2], mm[2], vv[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = threadIdx.x + k * THREADS;
            ww[k] = ((Four *)w)[i]; mm[k] = ((Four *)m)[i]; vv[k] = ((Four *)v)[i];
            const float4 x = __ldcs((const float4 *)g + i);
            gg[k] = Four{{x.x, x.y}, {x.z, x.w}};
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = threadIdx.x + k * THREADS;
            adamw_two(ww[k].lo, gg[k].lo, mm[k].lo, vv[k].lo, a, u);
            adamw_two(ww[k].hi, gg[k].hi, mm[k].hi, vv[k].hi, a, u);
            ((Four *)w)[i] = ww[k]; ((Four *)m)[i] = mm[k]; ((Four *)v)[i] = vv[k];
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

// The hash of a place and a step, its first line apart: eight neighbouring places from a multiple of eight on differ in it by their last three bits.
__device__ __forceinline__ unsigned random_seed(unsigned long long place, unsigned step) {
    return (unsigned)place ^ ((unsigned)(place >> 32) * 0x632BE5ABu) ^ (step * 0x9E3779B1u);
}
__device__ __forceinline__ unsigned random32(unsigned x) {
    x = (x ^ (x >> 16)) * 0xA3D95F4Bu;
    x = (x ^ (x >> 15)) * 0x6C8E9D73u;
    return x ^ (x >> 16);
}
// Two codes of m, from the places 2 k and 2 k + 1 of a word: with the exponent's bias of 7 that the conversion takes, 1.0 (the largest code there is) is
// 256 of its units.
__device__ __forceinline__ Two decode_m(unsigned word, int k, float top) {
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)(word >> (16 * k))));
    const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&h));
    return mul2(mul2(Two{f.x, f.y}, both(0x1p-8f)), both(top));
}
__device__ __forceinline__ Two decode_v(unsigned word, int k, float top) {
    const unsigned a = k ? word << 4 : word << 20, b = k ? word >> 4 : word << 12;
    return mul2(mul2(Two{__uint_as_float(a & 0x0ff00000u), __uint_as_float(b & 0x0ff00000u)}, both(1.f / V_UNIT)), both(top));
}
// An entry over the block's largest, in the units of the code, with the random bits added below the code's last place: the code is in the bits from 20
// on (at most the largest code: 1.0 has zeros below).
__device__ __forceinline__ Two scaled(Two x, float inv, float unit) { return mul2(mul2(x, both(inv)), both(unit)); }
__device__ __forceinline__ unsigned rounded(float x, unsigned random16) { return __float_as_uint(x) + (random16 << 4); }
// Byte 3 of each of four words
__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// A block whose largest entry is below the smallest normal float is held as zeros.  (Infinity times the smallest number is infinity still, whose bits give
// the largest code, and the finite entries beside it zeros.)
__device__ __forceinline__ float held(float x, float &inv) {
    if (x < 1.17549435e-38f) x = 0.f;
    inv = x > 0.f ? fmaxf(__frcp_rn(x), __uint_as_float(1u)) : 0.f;
    return x;
}

// A thread has EIGHT neighbouring entries, so eight threads share a block of 64.
constexpr int EIGHT = 8;
static_assert(CHUNK == EIGHT * THREADS, "one pass");
template <bool BOUNDED> __global__ void __launch_bounds__(THREADS) adamw8_kernel(const __grid_constant__ AdamWTable tab, const __grid_constant__ AdamWArgs by_value) {
    const int number = tensor_of(tab, blockIdx.x);
    const AdamWTensor &t = tab.t[number];
    const AdamWArgs a = adamw_args(tab, by_value, true);
    const Update u = update_of(a, tab.decay[number]);
    const long long at = (long long)(blockIdx.x - tab.first[number]) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.n - at), i = threadIdx.x * EIGHT;
    float *w = t.w + at + i;
    const float *g = t.g + at + i;
    char *block = (char *)t.m + (at + i) / BLOCK_ENTRIES * BLOCK_BYTES;
    uint2 *codes = (uint2 *)block + threadIdx.x % 8 * 2;
    const bool there = i / BLOCK_ENTRIES * BLOCK_ENTRIES < n;             // the tensor's last block may be short, its codes are there for all 64
    const bool whole = !(((uintptr_t)w | (uintptr_t)g) & 15) && i + EIGHT <= n;
    Two ww[4] = {}, gg[4] = {}, m[4], v[4];
    uint2 code[2] = {};
    float2 top = make_float2(0.f, 0.f);
    if (there) { code[0] = codes[0]; code[1] = codes[1]; top = *(const float2 *)(block + 128); }
    if (whole) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float4 x = ((const float4 *)w)[k], y = __ldcs((const float4 *)g + k);
            ww[2 * k] = Two{x.x, x.y}; ww[2 * k + 1] = Two{x.z, x.w};
            gg[2 * k] = Two{y.x, y.y}; gg[2 * k + 1] = Two{y.z, y.w};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (i + 2 * j < n) { ww[j].x = w[2 * j]; gg[j].x = g[2 * j]; }
            if (i + 2 * j + 1 < n) { ww[j].y = w[2 * j + 1]; gg[j].y = g[2 * j + 1]; }
        }
    }
    float am = 0.f, av = 0.f;                                 // a NaN is larger than all else, and its block shows it
#pragma unroll
    for (int j = 0; j < 4; j++) {
        m[j] = decode_m(code[j / 2].x, j % 2, top.x);
        v[j] = decode_v(code[j / 2].y, j % 2, top.y);
        adamw_two(ww[j], gg[j], m[j], v[j], a, u);
        if (!whole) {                                         // places behind the tensor's end
            if (i + 2 * j >= n) m[j].x = v[j].x = 0.f;
            if (i + 2 * j + 1 >= n) m[j].y = v[j].y = 0.f;
        }
        am = largest(am, largest(fabsf(m[j].x), fabsf(m[j].y)));
        av = largest(av, largest(v[j].x, v[j].y));
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        am = largest(am, __shfl_xor_sync(0xffffffffu, am, o));
        av = largest(av, __shfl_xor_sync(0xffffffffu, av, o));
    }
    float im, iv;
    const float lm = held(am, im), lv = held(av, iv);
    const unsigned least = BOUNDED && lv > 0.f && lv < __int_as_float(0x7f800000) ? 1u << 20 : 0u;         // the smallest code of v in its place
    const unsigned seed = random_seed((unsigned long long)(t.place + at + i), (unsigned)a.step);
    unsigned qm[8], qv[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned r0 = random32(seed ^ (2 * j)), r1 = random32(seed ^ (2 * j + 1));
        const Two sm = scaled(m[j], im, M_UNIT), sv = scaled(v[j], iv, V_UNIT);
        qm[2 * j] = rounded(sm.x, r0 & 0xffffu); qm[2 * j + 1] = rounded(sm.y, r1 & 0xffffu);
        qv[2 * j] = rounded(sv.x, r0 >> 16); qv[2 * j + 1] = rounded(sv.y, r1 >> 16);
        if (BOUNDED) {
            qv[2 * j] = max(qv[2 * j], v[j].x > 0.f ? least : 0u);
            qv[2 * j + 1] = max(qv[2 * j + 1], v[j].y > 0.f ? least : 0u);
        }
    }
    if (there) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const unsigned *x = qm + 4 * k, *y = qv + 4 * k;
            const unsigned size = top_bytes(x[0] << 4, x[1] << 4, x[2] << 4, x[3] << 4), sign = top_bytes(x[0], x[1], x[2], x[3]);
            codes[k] = make_uint2((size & 0x7f7f7f7fu) | (sign & 0x80808080u), top_bytes(y[0] << 4, y[1] << 4, y[2] << 4, y[3] << 4));
        }
        if (threadIdx.x % 8 == 0) *(float2 *)(block + 128) = make_float2(lm, lv);
    }
    if (whole) {
#pragma unroll
        for (int k = 0; k < 2; k++) ((float4 *)w)[k] = make_float4(ww[2 * k].x, ww[2 * k].y, ww[2 * k + 1].x, ww[2 * k + 1].y);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (i + 2 * j < n) w[2 * j] = ww[j].x;
            if (i + 2 * j + 1 < n) w[2 * j + 1] = ww[j].y;
        }
    }
}

__global__ void __launch_bounds__(256) adamw8_read_kernel(const char *__restrict__ state, float *__restrict__ m, float *__restrict__ v, long long n) {
    const bool vec = !(((uintptr_t)m | (uintptr_t)v) & 15);
    const long long p = (long long)blockIdx.x * 256 + threadIdx.x;
    if (p * 4 < n) {
        const char *blk = state + p / 16 * BLOCK_BYTES;
        const uint2 c = ((const uint2 *)blk)[p & 15];
        const float2 top = *(const float2 *)(blk + 128);
        const Two x0 = decode_m(c.x, 0, top.x), x1 = decode_m(c.x, 1, top.x), y0 = decode_v(c.y, 0, top.y), y1 = decode_v(c.y, 1, top.y);
        const float x[4] = {x0.x, x0.y, x1.x, x1.y}, y[4] = {y0.x, y0.y, y1.x, y1.y};
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

enum Form { IN_32, IN_8, IN_8_BOUNDED };
int adamw(Form form, int count, float *const *w, const float *const *g, void *const *m, float *const *v, const long long *n, const float *decay,
          const AdamWArgs &a, const float *hyper, long long first, const char *name) {
    SEERA_ENSURE();
    const bool eight = form != IN_32;
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
    const void *kernel = form == IN_32 ? (const void *)adamw_kernel : (form == IN_8 ? (const void *)adamw8_kernel<false> : (const void *)adamw8_kernel<true>);
    AdamWTable table;
    AdamWArgs args = a;
    for (int i = 0; i < count;) {
        memset(&table, 0, sizeof table);
        table.hyper = hyper;
        long long blocks = 0;
        for (; i < count && table.count < TABLE; i++) {
            if (n[i] == 0) continue;
            const long long need = (n[i] + CHUNK - 1) / CHUNK;
            if (blocks + need > 0x7fffffffLL) break;
            table.first[table.count] = (unsigned)blocks;
            table.decay[table.count] = decay[i];
            AdamWTensor &t = table.t[table.count++];
            t.w = w[i]; t.g = g[i]; t.m = m[i]; t.n = n[i];
            if (eight) t.place = first;
            else t.v = v[i];
            blocks += need;
            if (eight) first += (n[i] + BLOCK_ENTRIES - 1) / BLOCK_ENTRIES * BLOCK_ENTRIES;
        }
        if (!table.count) break;                              // tensors without entries were the last
        std::shared_ptr<void> kept;                           // a recorded launch's table, for other scalars
        if (rt().capturing && !hyper) {
            try {
                kept = std::make_shared<AdamWTable>(table);
            } catch (const std::bad_alloc &) {
                return fail(SEERA_E_OOM, "%s: no host memory", name);
            }
        }
        void *argv[] = {&table, &args};
        cudaLaunchKernel(kernel, dim3((unsigned)blocks), dim3(THREADS), argv, 0, rt().stream);
        SEERA_LAUNCH_CHECK(name);
        if (kept) {
            OptLaunch l = {};
            l.kind = 2; l.grid = (int)blocks; l.n_scalars = eight ? 10 : 9;
            memcpy(l.scalars, &args, sizeof(float) * l.n_scalars);
            l.func = kernel;
            l.table = kept;
            if (int s = graph_note_optimizer(l)) return s;
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
    return adamw(IN_32, count, w, g, (void *const *)m, v, n, decay, {lr, beta1, omb1, beta2, omb2, eps, c1, c2, grad_scale, 0.f}, hyper, 0,
                 "adamw_step");
}

size_t seera_adamw8_state_bytes(long long n) { return n < 0 ? 0 : (size_t)((n + BLOCK_ENTRIES - 1) / BLOCK_ENTRIES) * BLOCK_BYTES; }

int seera_adamw8_step(int count, float *const *w, const float *const *g, void *const *state, const long long *n, const float *decay, float lr,
                      float beta1, float omb1, float beta2, float omb2, float eps, float c1, float c2, float grad_scale, float step,
                      const float *hyper, long long first) {
    if (!(step >= 0.f && step < 4294967040.f) && !hyper) return fail(SEERA_E_ARG, "adamw8_step: step %g", (double)step);
    return adamw(IN_8, count, w, g, state, nullptr, n, decay, {lr, beta1, omb1, beta2, omb2, eps, c1, c2, grad_scale, step}, hyper, first,
                 "adamw8_step");
}
int seera_adamw8_bounded_step(int count, float *const *w, const float *const *g, void *const *state, const long long *n, const float *decay, float lr,
                              float beta1, float omb1, float beta2, float omb2, float eps, float c1, float c2, float grad_scale, float step,
                              const float *hyper, long long first) {
    if (!(step >= 0.f && step < 4294967040.f) && !hyper) return fail(SEERA_E_ARG, "adamw8_bounded_step: step %g", (double)step);
    return adamw(IN_8_BOUNDED, count, w, g, state, nullptr, n, decay, {lr, beta1, omb1, beta2, omb2, eps, c1, c2, grad_scale, step}, hyper, first,
                 "adamw8_bounded_step");
}

int seera_adamw8_read(const void *state, float *m, float *v, long long n) {
    SEERA_ENSURE();
    if (n < 0 || (n > 0 && (!state || !m || !v)) || ((uintptr_t)state & 7)) return fail(SEERA_E_ARG, "adamw8_read: bad argument");
    if (n > (1LL << 40)) return fail(SEERA_E_LIMIT, "adamw8_read: %lld entries", n);
    if (n == 0) return SEERA_OK;
    adamw8_read_kernel<<<(unsigned)((n + 1023) / 1024), 256, 0, rt().stream>>>((const char *)state, m, v, n);
    SEERA_LAUNCH_CHECK("adamw8_read");
    return SEERA_OK;
}

}  // extern "C"
