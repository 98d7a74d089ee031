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
#include "pairs.cuh"
#include "sigmoid.cuh"
#include "tc_ptx.cuh"
#include <initializer_list>

namespace seera {

int *tc_status_word();                                    // contraction_tc.cu

namespace {
struct Waits { int *status; unsigned long long clocks; };  // where a wait that runs out is noted, and its budget
struct ScanFwd {
    const float *f, *v, *h0;
    const int *lengths;
    float *h, *last;
    long long ld;
    int N, T, C, ranks;
    Waits waits;
};
struct ScanBwd {
    const float *f, *v, *h0;
    const int *lengths;
    const float *h, *dh, *dlast;
    float *df, *dv, *dh0;
    long long ld, ldg;
    int N, T, C, ranks;
    Waits waits;
};

// A gate is kept as sigmoid_less gives it, the smaller of a and 1 - a, which has its full relative precision, with the sign bit where that is a: a state that decays by
// 1e-4 a step is summed over ten thousand of them, and one minus a rounded a would have lost four of seven digits there.
constexpr float HOLD = 0.f;                               // the gate of a step that is not there: a = 1
__device__ __forceinline__ bool keeps(float s) { return __float_as_int(s) >= 0; }       // (the sign of a zero counts)
// a h + (1 - a) v = h + s (v - h) or v - s (v - h)
__device__ __forceinline__ float step_of(float s, float h, float v) { return fmaf(s, v - h, keeps(s) ? h : v); }
// a x and (1 - a) x
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
            if (t + k < len) s = step_of(sigmoid_less(ff[k]), s, vv[k]);
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
            const float gate = sigmoid_less(p.f[row * p.ld + c]), g = (p.dh ? p.dh[row * p.C + c] : 0.f) + s;
            const float before = t ? p.h[(row - 1) * p.C + c] : (p.h0 ? p.h0[i] : 0.f);
            part(gate, g, s, dv);
            df = (1.f - fabsf(gate)) * (fabsf(gate) * g) * (before - p.v[row * p.ld + c]);
        }
        p.df[row * p.ldg + c] = df;
        p.dv[row * p.ldg + c] = dv;
    }
    if (p.dh0) p.dh0[i] = s;
}

// ---- time split over half-warps, warps and the blocks of a cluster --------------------------------------------------------------------
// A lane has two neighbouring channels of a tile of 32 (half a warp reads whole lines, and pairs halve what is not arithmetic), a half-warp L neighbouring
// steps of them, a block W warps of those and the blocks of a cluster follow one another; the cluster then goes on to the next such piece of
// time.  What a run of steps does to a state is one multiply-add, x -> A x + B.  A thread forms it for each of its steps from its first one on; warps put
// theirs into shared memory, blocks send theirs to the others of the cluster; with the state at its start every step is one multiply-add more.
// A warp copies its own steps into its own part of shared memory, STAGES - 1 pieces ahead: nothing waits for another warp's data, and the loads
// cost neither registers nor, with 16 bytes a copy, more than a quarter of an instruction an element.  (A third stage gained nothing.)
// Between blocks the runs travel by stores that count their bytes on a barrier in the receiver's shared memory (a barrier of the cluster would wait for
// every result written before it); one warp sends and another takes in, since each warp that went through the other blocks' runs itself would read more
// of them from shared memory than data.  Two places are used in turn: who writes one for the second next piece has received everybody's run of the
// next one, which each sends after it has read the place.
// Measured (fp32, inputs beyond L2): forward of 8 x 2048 x 2048 78 us (5.2 TB/s, the bytes), of one sequence of 65536 x 512 93 us (4.3 TB/s; 13 blocks
// a tile, two an SM, leave a quarter of the SMs idle, and the others wait for one another's runs); backward of 8 x 2048 x 2048 148 us (5.4 TB/s).  With all
// warps sending and taking in the second took 108 us; a lane with one channel and 16 steps took 80, 137 and 148 us, a tile of 64 channels 102, 220 and 162.
// Rows that start anywhere, 7 x 1023 x 645 backward: 28 us, 39 with copies of single words, 76 with loads into registers.
constexpr int MAX_RANKS = 16, STAGES = 2, TILE = 32, WARPS = 8, FWD_STEPS = 8, BWD_STEPS = 4;

__device__ __forceinline__ Two pick(bool kx, bool ky, Two a, Two b) { return Two{kx ? a.x : b.x, ky ? a.y : b.y}; }
// sigmoid_less of two, bit for bit
__device__ __forceinline__ Two sigmoid_less2(Two f) {
    Two x, e, s;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x.x) : "f"(fabsf(f.x)), "f"(88.f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x.y) : "f"(fabsf(f.y)), "f"(88.f));
    const Two t = mul2(x, both(1.44269502f)), gone = fma2(x, both(-1.44269502f), t);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = fma2(e, mul2(gone, both(-0.693147182f)), e);
    e = add2(e, both(1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
    return Two{copysignf(s.x, f.x), copysignf(s.y, f.y)};
}

struct __align__(16) Run { Two a, b; };                   // x -> a x + b for each of a lane's channels
__device__ __forceinline__ Run no_steps() { return Run{both(1.f), both(0.f)}; }
__device__ __forceinline__ Two after(const Run &r, Two x) { return fma2(r.a, x, r.b); }
__device__ __forceinline__ Run then(const Run &first, const Run &second) { return Run{mul2(first.a, second.a), after(second, first.b)}; }
template <int W> struct Joined {
    Run warps[3][W][16], ranks[2][MAX_RANKS][16];
    Two carry[2][16];
    unsigned long long bar[2];
};

__device__ __forceinline__ void send(Run *place, unsigned long long *bar, int rank, const Run &v) {
    uint32_t to, done;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(place)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(done) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "f"(v.a.x), "f"(v.a.y), "f"(v.b.x),
                 "f"(v.b.y), "r"(done) : "memory");
}
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: a wait that runs out is noted, and the thread goes on without waiting any more (it still sends all it has to, and no block leaves early).
__device__ __forceinline__ void await(uint32_t bar, uint32_t parity, Waits &w) {
    if (arrived(bar, parity) || !w.clocks) return;
    const long long t0 = clock64();
    while (!arrived(bar, parity))
        if ((unsigned long long)(clock64() - t0) > w.clocks) {
            if (w.status) atomicCAS(w.status, 0, 5);
            w.clocks = 0;
            return;
        }
}
// A copy of 16 bytes from global into shared memory that the thread does not wait for.
__device__ __forceinline__ void copy_async(float *to, const float *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }

// Which channels, steps and sequence a thread has, and how its runs and those of others are joined.
// VEC: whether rows start on 16 bytes and hold whole ones.  Where they do not, the whole 16 bytes that hold a row's part of the tile are copied, up to three
// floats of what lies beside it with it (16 bytes that hold a float of a tensor belong to its allocation).
template <int W, int L, bool VEC> struct Place {
    static constexpr int STEPS = 2 * L;                    // of a warp
    // Floats from row to row in shared memory, those that keep the half-warps' rows on different banks, and those of a tensor that a warp copies of a piece
    static constexpr int WIDTH = VEC ? TILE : TILE + 4, GAP = VEC || L * WIDTH % 32 ? 0 : 16, ROWS = STEPS * WIDTH + GAP;
    // One lane has two neighbouring channels, or two that are 16 apart, which single words are read and written side by side with.
    static constexpr int APART = VEC ? 1 : 16;
    Joined<W> &sm;
    int warp, lane, half, col, in, rank, ranks, n, c0, c, len, piece, first;       // in: the place of the lane's first channel in its tile
    bool on, on2;                                          // whether the lane's channels are there
    Waits waits;
    Two carry;                                             // several blocks: the state at the start of the piece, in the warp that takes it in
    template <class P> __device__ __forceinline__ Place(const P &p, Joined<W> &sm_) : sm(sm_) {
        warp = threadIdx.x >> 5; lane = threadIdx.x & 31; half = lane >> 4; col = lane & 15; ranks = p.ranks; rank = blockIdx.x % ranks;
        const unsigned tiles = (p.C + TILE - 1) / TILE, tile = blockIdx.x / ranks;
        n = tile / tiles;
        c0 = (tile - n * tiles) * TILE;
        in = VEC ? 2 * col : col;
        c = c0 + in;
        on = c < p.C; on2 = c + APART < p.C;
        len = length_of(p.lengths, n, p.T);
        piece = ranks * W * STEPS;
        first = (rank * W + warp) * STEPS;
        waits = p.waits;
    }
    __device__ __forceinline__ Two state(const float *p, int C) const {
        const long long i = (long long)n * C + c;
        return Two{on && p ? p[i] : 0.f, on2 && p ? p[i + APART] : 0.f};
    }
    __device__ __forceinline__ void begin(Two x) {
        carry = x;
        if (ranks == 1) {
            if (threadIdx.x < 16) sm.carry[0][col] = x;    // (read behind the first piece's barrier)
            return;
        }
        if (threadIdx.x == 0) {
            mbar_init(smem_u32(&sm.bar[0]), 1);
            mbar_init(smem_u32(&sm.bar[1]), 1);
            fence_mbar_init();
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    // What the thread's steps of piece k do to a state (`run`): its warp's goes to shared memory, and `run` is then what the warp's other half does in
    // front of it.  A barrier of the block follows, then pass_on.
    __device__ __forceinline__ void give(int k, Run &run) {
        Run other;
        other.a = two(__shfl_xor_sync(0xffffffffu, bits(run.a), 16));
        other.b = two(__shfl_xor_sync(0xffffffffu, bits(run.b), 16));
        if (!half) sm.warps[k % 3][warp][col] = then(run, other);
        run = half ? other : no_steps();
    }
    // The block's steps of piece k, sent to every block of the cluster by one warp.
    __device__ __forceinline__ void pass_on(int k) {
        if (ranks == 1 || warp != 0) return;
        const int buf = k & 1;
        const Run *runs = &sm.warps[k % 3][0][col];
        Run all = runs[0];
#pragma unroll
        for (int i = 1; i < W; i++) all = then(all, runs[16 * i]);
        if (threadIdx.x == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&sm.bar[buf])), "r"(ranks * 16 * (int)sizeof(Run)) : "memory");
        for (int r = half; r < ranks; r += 2) send(&sm.ranks[buf][rank][col], &sm.bar[buf], r, all);
    }
    // The state at the start of the block's steps of piece k, put into shared memory by another warp.  A barrier of the block follows, then start.
    __device__ __forceinline__ void take_in(int k) {
        if (ranks == 1 || warp != 1) return;
        const int buf = k & 1;
        await(smem_u32(&sm.bar[buf]), (k >> 1) & 1, waits);
#pragma unroll 4
        for (int r = 0; r < rank; r++) carry = after(sm.ranks[buf][r][col], carry);
        if (!half) sm.carry[buf][col] = carry;
#pragma unroll 4
        for (int r = rank; r < ranks; r++) carry = after(sm.ranks[buf][r][col], carry);
    }
    // The state at the start of the thread's steps of piece k.
    __device__ __forceinline__ Two start(int k, const Run &before) {
        Two x = sm.carry[k & 1][col];
        const Run *runs = &sm.warps[k % 3][0][col];
#pragma unroll
        for (int i = 0; i < W - 1; i++)
            if (i < warp) x = after(runs[16 * i], x);
        if (ranks == 1 && warp == W - 1 && !half) sm.carry[(k + 1) & 1][col] = after(runs[16 * (W - 1)], x);
        return after(before, x);
    }
    // The state behind the last of k pieces goes to `last`.  No block leaves while another may still send to it: every block has waited for all
    // that is sent to it, which the cluster's barrier makes sure of where a wait has run out.
    __device__ __forceinline__ void end(int k, float *last, int C) {
        if (ranks == 1) __syncthreads();
        if (last && rank == 0 && warp == (ranks > 1) && !half) {
            if (ranks == 1) carry = sm.carry[k & 1][col];
            const long long i = (long long)n * C + c;
            if (on) last[i] = carry.x;
            if (on2) last[i + APART] = carry.y;
        }
        if (ranks == 1) return;
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }
    // Steps t0 .. t0 + STEPS - 1 of a tensor whose rows are `ld` floats apart into shared memory, those of them in [lo, len); `from`: where row t0 of
    // this sequence and the tile's first channel are.
    __device__ __forceinline__ void copy(float *to, const float *from, int t0, long long ld, int lo, int C) const {
        if constexpr (VEC) {
            constexpr int ACROSS = TILE / 4, DOWN = 32 / ACROSS;
            const int x = lane % ACROSS * 4, y = lane / ACROSS;
            if (c0 + x >= C) return;
            const float *p = from + y * ld + x;
            float *t = to + y * TILE + x;
            if (t0 >= lo && t0 + STEPS <= len) {
#pragma unroll
                for (int i = 0; i < STEPS; i += DOWN, p += DOWN * ld) copy_async(t + i * TILE, p);
            } else {
#pragma unroll
                for (int i = 0; i < STEPS; i += DOWN, p += DOWN * ld)
                    if (t0 + i + y >= lo && t0 + i + y < len) copy_async(t + i * TILE, p);
            }
        } else {
            constexpr int ACROSS = WIDTH / 4;
            const int width = min(TILE, C - c0);
#pragma unroll
            for (int i = 0; i < STEPS * ACROSS; i += 32) {
                const int y = (i + lane) / ACROSS, x = (i + lane) % ACROSS * 4;
                const float *p = from + y * ld;
                const int before = shift(p);
                if (y < STEPS && t0 + y >= lo && t0 + y < len && x < before + width) copy_async(row(to, y) + x, p - before + x);
            }
        }
    }
    __device__ __forceinline__ static int shift(const float *p) { return VEC ? 0 : (int)((uintptr_t)p >> 2 & 3); }
    __device__ __forceinline__ static float *row(float *rows, int y) { return rows + y * WIDTH + (y >= L ? GAP : 0); }
    // The lane's channels of the i-th of its half's L steps, where `shift` of that row is `before` (from: the half's first row), and to a row in global memory.
    __device__ __forceinline__ Two get(const float *from, int i, int before) const {
        const float *p = from + i * WIDTH + before + in;
        if (VEC) return *reinterpret_cast<const Two *>(p);
        return Two{p[0], p[APART]};
    }
    __device__ __forceinline__ void put(float *p, Two v) const {
        if (VEC) {
            __stcs(reinterpret_cast<float2 *>(p), make_float2(v.x, v.y));
        } else {
            __stcs(p, v.x);
            if (on2) __stcs(p + APART, v.y);
        }
    }
};

template <int W, int L, bool VEC> __global__ void __launch_bounds__(W * 32, 16 / W) scan_fwd_kernel(const __grid_constant__ ScanFwd p) {
    typedef Place<W, L, VEC> Me;
    constexpr int ROWS = Me::ROWS;
    __shared__ Joined<W> sm;
    extern __shared__ __align__(16) float stages[];         // [STAGES][W][f, v][2 L][TILE]
    Me me(p, sm);
    const long long at = (long long)me.n * p.T;
    float *mine = stages + me.warp * 2 * ROWS;
    auto request = [&](int t0, int stage) {
        float *to = mine + stage * W * 2 * ROWS;
        if (t0 < me.len) {
            me.copy(to, p.f + (at + t0) * p.ld + me.c0, t0, p.ld, 0, p.C);
            me.copy(to + ROWS, p.v + (at + t0) * p.ld + me.c0, t0, p.ld, 0, p.C);
        }
        copies_commit();
    };
    int t0 = me.first, stage = 0;
#pragma unroll
    for (int k = 0; k < STAGES - 1; k++) request(t0 + k * me.piece, k);
    me.begin(me.state(p.h0, p.C));
    const int own = me.half * L;                            // the thread's steps among the warp's
    auto work = [&](Run (&m)[L], int t0) {                  // the steps as one multiply-add each from the thread's first one on
        copies_wait();
        __syncwarp();                                       // the piece is there for every lane, and the stage before it is read
        request(t0 + (STAGES - 1) * me.piece, stage == 0 ? STAGES - 1 : stage - 1);
        const float *from = Me::row(mine + stage * W * 2 * ROWS, own);
        const float *pf = p.f + (at + t0 + own) * p.ld + me.c0, *pv = p.v + (at + t0 + own) * p.ld + me.c0;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        auto steps = [&](bool all) {
            Run run = no_steps();
#pragma unroll
            for (int i = 0; i < L; i++) {
                if (all || t0 + own + i < me.len) {
                    const Two f = me.get(from, i, Me::shift(pf + i * p.ld)), v = me.get(from + ROWS, i, Me::shift(pv + i * p.ld)), s = sigmoid_less2(f);
                    const bool kx = keeps(s.x), ky = keeps(s.y);
                    run.b = fma2(s, less2(v, run.b), pick(kx, ky, run.b, v));
                    run.a = fma2(Two{-s.x, -s.y}, run.a, pick(kx, ky, run.a, both(0.f)));
                }
                m[i] = run;
            }
        };
        if (t0 + Me::STEPS <= me.len) steps(true);
        else steps(false);
    };
    auto write = [&](const Run (&m)[L], Two x, int t0) {
        t0 += own;
        if (!p.h || !me.on || t0 >= p.T) return;
        float *h = p.h + (at + t0) * p.C + me.c;
        if (t0 + L <= me.len) {
#pragma unroll
            for (int i = 0; i < L; i++, h += p.C) me.put(h, after(m[i], x));
        } else {
#pragma unroll
            for (int i = 0; i < L; i++, h += p.C)
                if (t0 + i < p.T) me.put(h, t0 + i < me.len ? after(m[i], x) : both(0.f));
        }
    };
    int k = 0;
    Run before;
    auto go = [&](const Run (&now)[L], Run (&next)[L], bool more) {       // `now` has been worked on and its runs are passed on
        Run then_before;
        if (more) {
            work(next, t0 + me.piece);                      // (while the others' runs are on their way)
            then_before = next[L - 1];
            me.give(k + 1, then_before);
        }
        me.take_in(k);
        __syncthreads();
        if (more) me.pass_on(k + 1);
        write(now, me.start(k, before), t0);
        before = then_before;
        t0 += me.piece;
        k++;
    };
    Run one[L], two[L];
    work(one, t0);
    before = one[L - 1];
    me.give(0, before);
    __syncthreads();
    me.pass_on(0);
    for (long long start = 0; start < p.T; start += 2 * me.piece) {
        const bool more = start + me.piece < p.T;
        go(one, two, more);
        if (!more) break;
        go(two, one, start + 2 * me.piece < p.T);
    }
    me.end(k, p.last, p.C);
}

// Backward: the same with time running from the end, where c -> a (dh + c) is what a step does.
template <int W, int L, bool VEC> __global__ void __launch_bounds__(W * 32, 16 / W) scan_bwd_kernel(const __grid_constant__ ScanBwd p) {
    typedef Place<W, L, VEC> Me;
    constexpr int ROWS = Me::ROWS;
    __shared__ Joined<W> sm;
    extern __shared__ __align__(16) float stages[];         // [STAGES][W][f, v, dh, h of the step before][2 L][TILE]
    Me me(p, sm);
    const long long at = (long long)me.n * p.T;
    float *mine = stages + me.warp * 4 * ROWS;
    auto request = [&](int t0, int stage) {                 // steps t0 .. t0 + 2 L - 1, of which some may lie before the first
        float *to = mine + stage * W * 4 * ROWS;
        if (t0 + Me::STEPS > 0 && t0 < me.len) {
            me.copy(to, p.f + (at + t0) * p.ld + me.c0, t0, p.ld, 0, p.C);
            me.copy(to + ROWS, p.v + (at + t0) * p.ld + me.c0, t0, p.ld, 0, p.C);
            if (p.dh) me.copy(to + 2 * ROWS, p.dh + (at + t0) * p.C + me.c0, t0, p.C, 0, p.C);
            me.copy(to + 3 * ROWS, p.h + (at + t0 - 1) * p.C + me.c0, t0, p.C, 1, p.C);
        }
        copies_commit();
    };
    int t0 = p.T - me.first - Me::STEPS, stage = 0, k = 0;
#pragma unroll
    for (int k = 0; k < STAGES - 1; k++) request(t0 - k * me.piece, k);
    me.begin(me.state(p.dlast, p.C));
    const Two h0 = me.state(p.h0, p.C);
    const int own = (1 - me.half) * L;                      // the first half-warp has the later steps
    for (; k * (long long)me.piece < p.T; k++, t0 -= me.piece) {
        copies_wait();
        __syncwarp();
        request(t0 - (STAGES - 1) * me.piece, stage == 0 ? STAGES - 1 : stage - 1);
        const float *from = Me::row(mine + stage * W * 4 * ROWS, own);
        const float *pf = p.f + (at + t0 + own) * p.ld + me.c0, *pv = p.v + (at + t0 + own) * p.ld + me.c0;
        const float *pd = p.dh + (at + t0 + own) * p.C + me.c0, *ph = p.h + (at + t0 + own - 1) * p.C + me.c0;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        Two s[L], e[L], w[L];                               // gate, dh, h[t-1] - v[t]
        Run run = no_steps();
        auto work = [&](bool all) {
#pragma unroll
            for (int i = L - 1; i >= 0; i--) {
                const int t = t0 + own + i;
                s[i] = both(HOLD); e[i] = both(0.f); w[i] = both(0.f);
                if (all || (t >= 0 && t < me.len)) {
                    Two h = me.get(from + 3 * ROWS, i, Me::shift(ph + i * (long long)p.C));
                    if (!all && t == 0) h = h0;
                    s[i] = sigmoid_less2(me.get(from, i, Me::shift(pf + i * p.ld)));
                    w[i] = less2(h, me.get(from + ROWS, i, Me::shift(pv + i * p.ld)));
                    if (p.dh) e[i] = me.get(from + 2 * ROWS, i, Me::shift(pd + i * (long long)p.C));
                    const bool kx = keeps(s[i].x), ky = keeps(s[i].y);
                    const Two g = add2(e[i], run.b), ns = Two{-s[i].x, -s[i].y};
                    run.b = fma2(ns, g, pick(kx, ky, g, both(0.f)));
                    run.a = fma2(ns, run.a, pick(kx, ky, run.a, both(0.f)));
                }
            }
        };
        if (t0 > 0 && t0 + Me::STEPS <= me.len) work(true);
        else work(false);
        me.give(k, run);
        __syncthreads();
        me.pass_on(k);
        me.take_in(k);
        if (me.ranks > 1) __syncthreads();
        Two x = me.start(k, run);
        const int t1 = t0 + own;
        if (me.on && t1 + L > 0) {
            float *pf = p.df + (at + t1 + L - 1) * p.ldg + me.c, *pv = p.dv + (at + t1 + L - 1) * p.ldg + me.c;
            auto write = [&](bool all) {
#pragma unroll
                for (int i = L - 1; i >= 0; i--, pf -= p.ldg, pv -= p.ldg) {
                    const int t = t1 + i;
                    if (!all && t < 0) break;
                    const Two as = Two{fabsf(s[i].x), fabsf(s[i].y)}, g = add2(e[i], x), y = mul2(as, g), z = less2(g, y);
                    const bool kx = keeps(s[i].x), ky = keeps(s[i].y);
                    x = pick(kx, ky, z, y);
                    Two dv = pick(kx, ky, y, z), df = mul2(mul2(less2(both(1.f), as), y), w[i]);
                    if (!all && t >= me.len) dv = df = both(0.f);
                    me.put(pf, df);
                    me.put(pv, dv);
                }
            };
            if (t1 >= 0 && t1 + L <= me.len) write(true);
            else write(false);
        }
    }
    me.end(k, p.dh0, p.C);
}

// Clusters of each size that are resident at once (0: not asked yet), as the device's groups of SMs and the kernel's resources allow.
struct Resident { int clusters[MAX_RANKS + 1]; };
// Blocks of a cluster: every cluster works through its tile's pieces one after the other, and the clusters that are not resident at once follow in
// further rounds; the fewest pieces in a row win, and of equal sizes the smallest.  One sequence of 65536 steps and 512 channels, 16 tiles: 13 blocks take
// 93 us; with every warp taking part in the exchange 13 took 111, 8 took 151, and 16, of which 14 clusters are resident, 145.
// A block a tile where that leaves no place idle, whatever the count of pieces says: a cluster's blocks begin and end together and wait for one another.  512
// sequences of 192 x 1024 take 329 us forward and 433 backward with one block, 513 forward with two; of 96 backward 304 and 503; 64 of 256 x 512 32 and 40 forward.  With few
// tiles clusters win: 7 of 1024 x 645 backward 36 us, 41 with one block.
template <int W, class P> int launch_scan(void (*kernel)(P), Resident &known, P p, int steps, int rows, const char *name) {
    const long long tiles = (long long)p.N * ((p.C + TILE - 1) / TILE);
    const size_t smem = (size_t)STAGES * W * rows * sizeof(float);
    if (int s = check_cuda(allow_smem((const void *)kernel, smem), name)) return s;
    // (more than 8 is not promised on every device)
    if (!known.clusters[1]) {
        if (int s = check_cuda(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), name)) return s;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.blockDim = dim3(W * 32); cfg.dynamicSmemBytes = smem; cfg.stream = rt().stream; cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    long long least = 0;
    for (int r = 1; r <= MAX_RANKS; r++) {
        if (r > 1 && tiles >= known.clusters[1]) break;
        int &resident = known.clusters[r];
        if (!resident) {
            attr[0].val.clusterDim.x = (unsigned)r; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3((unsigned)r); cfg.numAttrs = 1;
            int most = 0;
            if (int s = check_cuda(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg), name)) return s;
            resident = most > 0 ? most : -1;
        }
        if (resident < 0 || tiles * r > 0x7fffffffLL) continue;
        const long long row = ((tiles + resident - 1) / resident) * ((p.T + (long long)r * W * steps - 1) / ((long long)r * W * steps));
        if (!least || row < least) { least = row; p.ranks = r; }
    }
    if (!least) return fail(SEERA_E_LIMIT, "%s: no block fits", name);
    p.waits = Waits{p.ranks > 1 ? tc_status_word() : nullptr, rt().tc_wait_clocks};
    if (p.ranks > 1) rt().tc_used = true;
    cfg.gridDim = dim3((unsigned)(tiles * p.ranks));
    attr[0].val.clusterDim.x = (unsigned)p.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = p.ranks > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return check_cuda(e, name);
    SEERA_LAUNCH_CHECK(name);
    return SEERA_OK;
}
bool on16(std::initializer_list<const void *> ps) {
    for (const void *p : ps) if (!aligned16(p)) return false;
    return true;
}
bool on8(std::initializer_list<const void *> ps) {
    for (const void *p : ps) if ((uintptr_t)p & 7) return false;
    return true;
}
// A padded batch with zeros behind each sequence's length; what is there is not read.  A sequence's floats in a row, so that a place is behind the length where it is not
// below length x C: bytes bound it (read and written once).
template <bool VEC> __global__ void __launch_bounds__(256) pad_steps_kernel(const float *x, const int *__restrict__ lengths, float *y, int N, int T, int C) {
    constexpr int V = VEC ? 4 : 1;
    const long long all = (long long)T * C, step = (long long)gridDim.x * 256 * V;
    for (int n = blockIdx.y; n < N; n += gridDim.y) {
        const long long live = (long long)length_of(lengths, n, T) * C;
        const float *from = x + n * all;
        float *to = y + n * all;
        for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < all; i += step) {
            if (VEC && i + V <= live) {
                *reinterpret_cast<float4 *>(to + i) = *reinterpret_cast<const float4 *>(from + i);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) to[i + j] = i + j < live ? from[i + j] : 0.f;
            }
        }
    }
}
// Whether the steps are few enough for a thread a state.  Those go at 0.27 us a step forward and 0.65 backward (two loads one after the other), and at the bytes' rate where states are many; the
// split form takes what a round of its blocks takes, 2.4 us, two blocks an SM and a tile each, however few the steps of its first piece are.  So up to STEPS steps a round,
// 9 forward and 4 backward; below a round's tenth the launch is all there is.  Thread a state against split, us forward / backward: 1 x 512 4 steps 7.1 / 8.2 against
// 7.3 / 7.2, 16 steps 10 / 15 against 7 / 7; 8 x 2048 8 steps 9.1 / 11.3 against 11.3 / 11.2, 32 steps 15 / 28 against 11 / 11; 64 x 1024 16 steps 11 / 19 against
// 22 / 24, 64 steps 28 / 56 against 27 / 32; 256 x 2048 16 steps 26 / 46 against 125 / 138, 64 steps 79 / 153 against 151 / 180.
template <int STEPS> bool few_steps(int N, int T, int C, int at_least) {
    const long long tiles = (long long)N * ((C + TILE - 1) / TILE);
    return T <= at_least || T <= STEPS * tiles / (2 * rt().sm_count);
}
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
    const ScanFwd p{gate, cand, h0, lengths, h, h_last, ld, N, T, C, 1, {}};
    ProfBytes pb((8.0 + (h ? 4 : 0)) * N * T * C, "gated_scan_fwd");
    if (few_steps<9>(N, T, C, 4)) {
        scan_fwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
        SEERA_LAUNCH_CHECK("gated_scan_fwd");
        return SEERA_OK;
    }
    const bool wide = C % 4 == 0 && ld % 4 == 0 && on16({gate, cand}) && on8({h});
    static Resident known[2];
    if (wide) return launch_scan<WARPS>(scan_fwd_kernel<WARPS, FWD_STEPS, true>, known[1], p, 2 * FWD_STEPS, 2 * Place<WARPS, FWD_STEPS, true>::ROWS, "gated_scan_fwd");
    return launch_scan<WARPS>(scan_fwd_kernel<WARPS, FWD_STEPS, false>, known[0], p, 2 * FWD_STEPS, 2 * Place<WARPS, FWD_STEPS, false>::ROWS, "gated_scan_fwd");
}

int seera_gated_scan_bwd(const float *gate, const float *cand, int ld, const float *h0, const int *lengths, const float *h, const float *dh,
                         const float *dh_last, float *dgate, float *dcand, int ld_grad, float *dh0, int N, int T, int C) {
    SEERA_ENSURE();
    if (N < 0 || T < 0 || C < 1 || ld < C || ld_grad < C || (N > 0 && T > 0 && (!gate || !cand || !h || !dgate || !dcand)) || (!dh && !dh_last))
        return fail(SEERA_E_ARG, "gated_scan_bwd: bad argument");
    if ((long long)N * C > 0x7fffffffLL || T > (1 << 30)) return fail(SEERA_E_LIMIT, "gated_scan_bwd: %lld states, %d steps", (long long)N * C, T);
    if (N == 0) return SEERA_OK;
    const ScanBwd p{gate, cand, h0, lengths, h, dh, dh_last, dgate, dcand, dh0, ld, ld_grad, N, T, C, 1, {}};
    ProfBytes pb((20.0 + (dh ? 4 : 0)) * N * T * C, "gated_scan_bwd");
    if (few_steps<4>(N, T, C, 2)) {
        scan_bwd_serial_kernel<<<(unsigned)(((long long)N * C + 127) / 128), 128, 0, rt().stream>>>(p);
        SEERA_LAUNCH_CHECK("gated_scan_bwd");
        return SEERA_OK;
    }
    const bool wide = C % 4 == 0 && ld % 4 == 0 && ld_grad % 2 == 0 && on16({gate, cand, h, dh}) && on8({dgate, dcand});
    static Resident known[2];
    if (wide) return launch_scan<WARPS>(scan_bwd_kernel<WARPS, BWD_STEPS, true>, known[1], p, 2 * BWD_STEPS, 4 * Place<WARPS, BWD_STEPS, true>::ROWS, "gated_scan_bwd");
    return launch_scan<WARPS>(scan_bwd_kernel<WARPS, BWD_STEPS, false>, known[0], p, 2 * BWD_STEPS, 4 * Place<WARPS, BWD_STEPS, false>::ROWS, "gated_scan_bwd");
}

int seera_pad_steps(const float *x, const int *lengths, float *y, int N, int T, int C) {
    SEERA_ENSURE();
    const long long all = (long long)T * C;
    if (N < 0 || T < 0 || C < 1 || (N > 0 && T > 0 && (!x || !lengths || !y))) return fail(SEERA_E_ARG, "pad_steps: bad argument");
    if (N == 0 || T == 0) return SEERA_OK;
    ProfBytes pb(8.0 * N * all, "pad_steps");
    const bool wide = all % 4 == 0 && on16({x, y});
    const int deep = N < 65535 ? N : 65535;
    const long long need = (all + (wide ? 1023 : 255)) / (wide ? 1024 : 256), most = (long long)rt().sm_count * 8 / deep + 1;
    const dim3 grid((unsigned)(need < most ? need : most), (unsigned)deep);
    if (wide) pad_steps_kernel<true><<<grid, 256, 0, rt().stream>>>(x, lengths, y, N, T, C);
    else pad_steps_kernel<false><<<grid, 256, 0, rt().stream>>>(x, lengths, y, N, T, C);
    SEERA_LAUNCH_CHECK("pad_steps");
    return SEERA_OK;
}

}  // extern "C"
