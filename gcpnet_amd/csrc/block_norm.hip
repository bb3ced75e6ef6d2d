// The norms before and after a residual block with its gate and residual scale, forward and backward:
//
//   u = post(y);  s = x + scale * act(gate) * u;  h = pre(s)              post, pre: layer norm, RMS norm or none
//
//   n2 = (s - mean2) rstd2;  gs = ds + rstd2 (dh w - mean(dh w) - n2 mean(dh w n2))      (RMS: without the mean)
//   dx = gs;  du = scale act(gate) gs;  dgate = scale gs u act'(gate);  dy = rstd1 (du w - mean(du w) - n1 mean(du w n1))
//   weights and biases: column sums of dh n2, dh, du n1, du, and of dgate for a gate of one value per channel.
//
// Bound: HBM -- forward reads x, y (and an element-wise gate) and writes s, h; backward reads x, y, ds, dh, writes dx, dy (s is formed
// again from x as the forward formed it, unrounded, for the same bytes that reading it would take).  A row is held in the registers of
// a group of 8 to 1024 threads between its reductions, so everything is read once; the statistics take two passes over the registers
// (mean, then squares of the differences).  The backward's groups walk many rows and keep the column sums in registers; one partial sum
// per workgroup goes through memory, summed in a fixed order by a second launch.
//
// 16384 x 4096 bf16, an element-wise gate, RMS norms: both directions 367 us for 1745 MB (4.7 TB/s, as a copy).  Its kernels, the median of 24
// in two runs: forward 123 - 125 us, backward 256 - 264 us (eight streams, and two sums over each row that all of its threads wait for); a norm alone 58 us.
#include <type_traits>

#include "elem_types.h"
#include "linear_tiles.h"

namespace {

constexpr int MAX_D = 16384, SETS = 5;  // sets of column sums: pre_w, post_w, pre_b, post_b, gate

struct NormArgs {
    int64_t rows;
    int d;
    const void *x, *y, *gate;
    int64_t x_ld, y_ld, gate_ld;  // gate_ld 0: one value per channel
    const void *post_w, *post_b, *pre_w, *pre_b;
    int post, pre, act, w_f32;
    float scale, slope, eps, inv_d;
    void *s, *h;
    float* stats;  // [rows, 4]: mean and 1 / sd of post, of pre
    const void *ds, *dh;
    void *dx, *dy, *dgate;
    float* part;  // [blocks, sets, d]
    int slot[SETS], sets;
    int held;  // the backward keeps the parameters in LDS
    int once, once_x, once_y;  // the forward's rows begin at 16 bytes; those of x and y are rows of their own
};
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));

// The waves of a workgroup meet and see each other's LDS writes.  (__syncthreads also waits for the wave's global loads and stores: for the row
// that was requested ahead, and for s to arrive in memory.)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Sums of K values over the G threads of a group; every thread gets them.  Groups of more than a wave exchange through LDS, in two
// buffers in turn, so that one barrier a call is enough.
template <int G, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float (*lds)[2][16], int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int d = (G < 64 ? G : 64) / 2; d; d >>= 1) v[k] += __shfl_xor(v[k], d);
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[turn][k][wave] = v[k];
        lds_barrier();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < G / 64; ++w) t += lds[turn][k][threadIdx.x / G * (G / 64) + w];
            v[k] = t;
        }
        turn ^= 1;
    }
}

// Rows that are read once, past the caches, where the parameters then stay (`once`, with an element-wise gate: 16384 x 4096 bf16 127 us a call against
// 138, 60000 x 1000 fp16 106 against 113, 16384 x 2048 fp32 106 against 125; a norm alone is at the rate of memory either way).  Not where rows begin off 16 bytes: a cache line is then asked for more than once (30000 x 1001: 66 us against 58).
// Nor one row that stands for all of them (x or y expanded): every group reads it again (16384 x 4096 bf16 84 us against 86, 16384 x 2048 fp32 64
// against 69).
template <class E, int V>
__device__ __forceinline__ Raw<E, V> row_load(const void* base, int64_t at, int count, bool once) {
    if (count == V && once) {
        const u32x4v x = __builtin_nontemporal_load((const u32x4v*)((const typename E::type*)base + at));
        return Raw<E, V>{{x[0], x[1], x[2], x[3]}};
    }
    return elem_load<E, V>(base, at, count);
}

template <class E, int G, int NV>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_fwd_kernel(NormArgs a) {
    constexpr int V = E::vec;
    constexpr int PER = (G > 256 ? G : 256) / G;  // groups of a workgroup
    __shared__ float lds[2][2][16];
    int turn = 0;
    const int t = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
    const bool on = row < a.rows;  // (a group of 256 or more is one workgroup: its rows are all on)
    const int64_t r = on ? row : 0;
    float u[NV][V], s[NV][V];
    int in[NV];  // elements of the row in the thread's vectors
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int left = a.d - (k * G + t) * V;
        in[k] = left < 0 ? 0 : left < V ? left : V;
    }
    Raw<E, V> xr[NV], yr[NV], gr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * G + t) * V;
        xr[k] = row_load<E, V>(a.x, r * a.x_ld + c, in[k], a.once_x);
        if (a.y) yr[k] = row_load<E, V>(a.y, r * a.y_ld + c, in[k], a.once_y);
        else yr[k] = elem_zero<E, V>();
        if (a.gate) gr[k] = row_load<E, V>(a.gate, r * a.gate_ld + c, in[k], a.once && a.gate_ld);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) u[k][j] = yr[k][j];
    float st[4] = {0.f, 1.f, 0.f, 1.f};
    auto normalize = [&](float (&z)[NV][V], int kind, float& mean, float& rstd) {  // z -> (z - mean) rstd
        if (kind == GCP_NORM_LAYER) {
            float v[1] = {0.f};
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) v[0] += z[k][j];  // (0 outside)
            group_sum<G, 1>(v, lds, turn);
            mean = v[0] * a.inv_d;
        }
        float q[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                z[k][j] = j < in[k] ? z[k][j] - mean : 0.f;
                q[0] += z[k][j] * z[k][j];
            }
        group_sum<G, 1>(q, lds, turn);
        rstd = 1.f / sqrtf(q[0] * a.inv_d + a.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) z[k][j] *= rstd;
    };
    if (a.post) normalize(u, a.post, st[0], st[1]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
        const int c = (k * G + t) * V;
        if (a.post_w) param_load<E, V>(a.post_w, c, in[k], a.w_f32).unpack(a.w_f32, w);
        if (a.post_b) param_load<E, V>(a.post_b, c, in[k], a.w_f32).unpack(a.w_f32, b);
        if (a.post)
#pragma unroll
            for (int j = 0; j < V; ++j) u[k][j] = fmaf(u[k][j], w[j], b[j]);
        if (a.gate) {
            float g[V], none[V];
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = gr[k][j];
            elem_act<V, false>(a.act, a.slope, g, g, none);
#pragma unroll
            for (int j = 0; j < V; ++j) u[k][j] *= g[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s[k][j] = j < in[k] ? (a.y ? fmaf(a.scale, u[k][j], xr[k][j]) : xr[k][j]) : 0.f;
        if (on && a.s) elem_store<E, V>(a.s, r * a.d + c, s[k], in[k]);
    }
    if (a.pre) {
        normalize(s, a.pre, st[2], st[3]);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V;
            float w[V], b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            if (a.pre_w) param_load<E, V>(a.pre_w, c, in[k], a.w_f32).unpack(a.w_f32, w);
            if (a.pre_b) param_load<E, V>(a.pre_b, c, in[k], a.w_f32).unpack(a.w_f32, b);
#pragma unroll
            for (int j = 0; j < V; ++j) s[k][j] = fmaf(s[k][j], w[j], b[j]);
            if (on) elem_store<E, V>(a.h, r * a.d + c, s[k], in[k]);
        }
    }
    if (a.stats && on && t == 0) *(f32x4*)(a.stats + 4 * r) = f32x4{st[0], st[1], st[2], st[3]};
}

// Waves per SIMD that the backward's registers leave room for; its workgroups are counted by them.
template <class E, int G, int NV>
constexpr int backward_waves() { return G > 512 ? 4 : NV > 1 ? 2 : E::vec == 8 ? 3 : 4; }
template <class E, int G, int NV>
constexpr int backward_groups() { return backward_waves<E, G, NV>() * 256 / (G > 256 ? G : 256); }  // of a CU
// Sets of column sums in registers: all, or with the rest in LDS, where there is room for it.
template <class E, int G, int NV>
constexpr int backward_kept() { return (G > 256 ? G : 256) * NV * E::vec * 12 <= 98304 ? 2 : SETS; }
// LDS of the backward, besides the parameters
template <class E, int G, int NV>
constexpr int backward_lds(bool bias) {
    return 256 + (G < 256 ? 256 * NV * E::vec * 4 : 16) + (bias && backward_kept<E, G, NV>() == 2 ? 3 * NV * E::vec * 4 * (G > 256 ? G : 256) : 16);
}

// BIAS: with the sums of the biases and of a gate of one value per channel, too.  Those lie in LDS, where each thread adds to places of its
// own: in registers they would take the room of the row that is requested ahead.
template <class E, int G, int NV, bool BIAS>
__global__ __launch_bounds__(G > 256 ? G : 256, E::vec == 8 && NV == 1 ? 3 : 1) void norm_bwd_kernel(NormArgs a) {
    constexpr int V = E::vec;
    constexpr int PER = (G > 256 ? G : 256) / G;
    // A gate's sigmoid is kept between its two uses where two workgroups a CU leave registers for it (16384 x 4096 bf16, both
    // directions: 407 us against 418), and formed twice where three are to fit (60000 x 1000 fp16, backward: 275 us against 286; three fit
    // with 168 registers: 249 us, with 170 two do: 354).
    constexpr bool KEEP = NV > 1;
    __shared__ float lds[2][2][16];
    __shared__ float cols[PER > 1 ? 256 * NV * V : 1];
    int turn = 0;
    const int t = threadIdx.x % G;
    int in[NV];  // elements of the row in the thread's vectors
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int left = a.d - (k * G + t) * V;
        in[k] = left < 0 ? 0 : left < V ? left : V;
    }
    constexpr int T = G > 256 ? G : 256, KEPT = backward_kept<E, G, NV>();
    __shared__ f32x4 more[BIAS && KEPT == 2 ? 3 * NV * (V / 4) * T : 1];
    float sum[BIAS ? KEPT : 2][NV][V];
    auto add = [&](int q, int k, const float (&v)[V]) {  // to a set of BIAS
        if constexpr (KEPT == 2) {
#pragma unroll
            for (int h = 0; h < V; h += 4) more[((q - 2) * NV + k) * (V / 4) * T + h / 4 * T + threadIdx.x] += f32x4{v[h], v[h + 1], v[h + 2], v[h + 3]};
        } else if constexpr (BIAS) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[q][k][j] += v[j];
        }
    };
    if constexpr (BIAS && KEPT == 2)
#pragma unroll
        for (int i = 0; i < 3 * NV * (V / 4); ++i) more[i * T + threadIdx.x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < (BIAS ? KEPT : 2); ++q)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[q][k][j] = 0.f;
    // post_w, post_b, pre_w, for all rows
    extern __shared__ u32x4v held[];
    constexpr int WORDS = V / 4;  // 16-byte words of a vector of fp32 parameters
    const bool wide = E::code != GCP_TYPE_F32 && a.w_f32;
    const int set = NV * G * (wide ? WORDS : 1);
    if (a.held) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const void* from = q == 0 ? a.post_w : q == 1 ? a.post_b : a.pre_w;
            if (from)
                for (int i = threadIdx.x; i < NV * G; i += T) {
                    const Param<E, V> v = param_load<E, V>(from, i * V, a.d - i * V < V ? a.d - i * V : V, a.w_f32);
                    held[q * set + i] = u32x4v{v.u[0], v.u[1], v.u[2], v.u[3]};
                    if constexpr (V == 8)
                        if (wide) held[q * set + NV * G + i] = u32x4v{v.u[4], v.u[5], v.u[6], v.u[7]};
                }
        }
        __syncthreads();
    }
    auto param = [&](int q, int k, float (&f)[V]) {
        const void* from = q == 0 ? a.post_w : q == 1 ? a.post_b : a.pre_w;
        if (!from) return;
        Param<E, V> v;
        if (a.held) {
            const u32x4v x = held[q * set + k * G + t];
            u32x4v y = {0u, 0u, 0u, 0u};
            if constexpr (V == 8)
                if (wide) y = held[q * set + NV * G + k * G + t];
#pragma unroll
            for (int j = 0; j < V; ++j) v.u[j] = j < 4 ? x[j & 3] : y[j & 3];
        } else {
            v = param_load<E, V>(from, (k * G + t) * V, in[k], a.w_f32);
        }
        v.unpack(a.w_f32, f);
    };
    const bool channel = a.gate && a.gate_ld == 0, full = KEEP && a.d == G * NV * V;  // (full: no thread has less than its vectors)
    struct Row { Raw<E, V> x[NV], y[NV], g[NV], ds[NV], dh[NV]; f32x4 st; };
    auto request = [&](int64_t first, Row& q) {
        const int64_t r = first + threadIdx.x / G;
        const bool on = r < a.rows;
        q.st = f32x4{0.f, 1.f, 0.f, 1.f};
        if (on && a.stats) q.st = *(const f32x4*)(a.stats + 4 * r);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V, n = on ? in[k] : 0;
            q.y[k] = a.y ? elem_load<E, V>(a.y, r * a.y_ld + c, n) : elem_zero<E, V>();
            q.x[k] = a.pre ? elem_load<E, V>(a.x, r * a.x_ld + c, n) : elem_zero<E, V>();
            q.g[k] = a.gate ? elem_load<E, V>(a.gate, r * a.gate_ld + c, n) : elem_zero<E, V>();
            q.ds[k] = a.ds ? elem_load<E, V>(a.ds, r * a.d + c, n) : elem_zero<E, V>();
            q.dh[k] = a.dh ? elem_load<E, V>(a.dh, r * a.d + c, n) : elem_zero<E, V>();
        }
    };
    // Waits for the row ahead at the end of a turn, before the turn's last stores: left to itself the compiler, which cannot count the loads
    // behind the branches, waits for all of them in front of the next turn's first use, those just requested included.
    auto arrived = [&](Row& q) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                asm volatile("" : "+v"(q.x[k].u[j]), "+v"(q.y[k].u[j]), "+v"(q.g[k].u[j]), "+v"(q.ds[k].u[j]), "+v"(q.dh[k].u[j])::"memory");
        asm volatile("" : "+v"(q.st)::"memory");
    };
    // (all groups of a workgroup make the same number of turns: barriers and shuffles stay in step.  AHEAD: a row is requested one turn
    // ahead, where the registers allow it)
    constexpr bool AHEAD = G <= 512;
    const int64_t step = (int64_t)gridDim.x * PER;
    Row ahead;
    if constexpr (AHEAD) {
        request((int64_t)blockIdx.x * PER, ahead);
        arrived(ahead);
    }
    for (int64_t first = (int64_t)blockIdx.x * PER; first < a.rows; first += step) {
        const int64_t row = first + threadIdx.x / G;
        const bool on = row < a.rows;
        const int64_t r = on ? row : 0;
        Row now;
        if constexpr (AHEAD) {
            now = ahead;
            request(first + step, ahead);
        } else {
            request(first, now);
        }
        const auto &xr = now.x, &yr = now.y, &gr = now.g, &dsr = now.ds, &dhr = now.dh;
        const f32x4 st = now.st;
        float gs[NV][V], sig[KEEP ? NV : 1][V];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) gs[k][j] = dsr[k][j];
        if (KEEP && a.gate && elem_by_sigmoid(a.act))
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) sig[k][j] = elem_sigmoid(gr[k][j]);
        if (a.dh) {
            float m[2] = {0.f, 0.f}, n2[NV][V], dn[NV][V];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (a.y) {  // s, as in the forward
                    float u[V], g[V], none[V], w[V], b[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; g[j] = gr[k][j]; u[j] = yr[k][j]; }
                    if (a.post) {
                        param(0, k, w);
                        param(1, k, b);
#pragma unroll
                        for (int j = 0; j < V; ++j) u[j] = fmaf((u[j] - st[0]) * st[1], w[j], b[j]);
                    }
                    if (a.gate) {
                        if constexpr (KEEP) elem_act_with<V, false>(a.act, a.slope, g, sig[k], g, none);
                        else elem_act<V, false>(a.act, a.slope, g, g, none);
#pragma unroll
                        for (int j = 0; j < V; ++j) u[j] *= g[j];
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) n2[k][j] = (fmaf(a.scale, u[j], xr[k][j]) - st[2]) * st[3];
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) n2[k][j] = (xr[k][j] - st[2]) * st[3];
                }
                float w[V], d[V];
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = 1.f;
                param(2, k, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    d[j] = dhr[k][j];  // (0 outside)
                    dn[k][j] = d[j] * w[j];
                    m[0] += dn[k][j];
                    m[1] = fmaf(dn[k][j], n2[k][j], m[1]);
                    sum[0][k][j] = fmaf(d[j], n2[k][j], sum[0][k][j]);
                }
                if constexpr (BIAS)
                    if (a.slot[2] >= 0) add(2, k, d);
            }
            group_sum<G, 2>(m, lds, turn);
            const float m0 = a.pre == GCP_NORM_LAYER ? m[0] * a.inv_d : 0.f, m1 = m[1] * a.inv_d;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) gs[k][j] = fmaf(st[3], fmaf(-n2[k][j], m1, dn[k][j] - m0), gs[k][j]);
        }
        if (a.dx)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (on) elem_store<E, V>(a.dx, r * a.d + (k * G + t) * V, gs[k], in[k]);
        if (!a.y) {
            if constexpr (AHEAD) arrived(ahead);
            continue;
        }
        float m[2] = {0.f, 0.f};  // (gs becomes du)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V;
            float w[V], b[V], n[V];
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            param(0, k, w);
            param(1, k, b);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                n[j] = (yr[k][j] - st[0]) * st[1];
                gs[k][j] = full || j < in[k] ? gs[k][j] * a.scale : 0.f;
            }
            if (a.gate) {
                float g[V], da[V];
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = gr[k][j];
                if constexpr (KEEP) elem_act_with<V, true>(a.act, a.slope, g, sig[k], g, da);
                else elem_act<V, true>(a.act, a.slope, g, g, da);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = a.post ? fmaf(n[j], w[j], b[j]) : yr[k][j];
                    da[j] *= gs[k][j] * u;
                    gs[k][j] *= g[j];
                }
                if constexpr (BIAS)
                    if (a.slot[4] >= 0) add(4, k, da);
                if (a.dgate && !channel && on) elem_store<E, V>(a.dgate, r * a.d + c, da, in[k]);
            }
            if constexpr (BIAS)
                if (a.slot[3] >= 0) add(3, k, gs[k]);
            if (a.post)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sum[1][k][j] = fmaf(gs[k][j], n[j], sum[1][k][j]);
                    gs[k][j] *= w[j];
                    m[0] += gs[k][j];
                    m[1] = fmaf(gs[k][j], n[j], m[1]);
                }
        }
        if (a.post) {
            group_sum<G, 2>(m, lds, turn);
            const float m0 = a.post == GCP_NORM_LAYER ? m[0] * a.inv_d : 0.f, m1 = m[1] * a.inv_d;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float n = (yr[k][j] - st[0]) * st[1];
                    gs[k][j] = st[1] * fmaf(-n, m1, gs[k][j] - m0);
                }
        }
        if constexpr (AHEAD) arrived(ahead);
        if (a.dy)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (on) elem_store<E, V>(a.dy, r * a.d + (k * G + t) * V, gs[k], in[k]);
    }
    // column sums: over the groups of the workgroup through LDS, then one partial row of each set that is wanted
#pragma unroll
    for (int q = 0; q < (BIAS ? SETS : 2); ++q) {
        if (a.slot[q] < 0) continue;  // (uniform)
        float* out = a.part + ((int64_t)blockIdx.x * a.sets + a.slot[q]) * a.d;
        if constexpr (PER > 1) __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int h = 0; h < V; h += 4) {
                f32x4 v;
                if constexpr (KEPT == 2) {
                    if (q < 2) v = f32x4{sum[q & 1][k][h], sum[q & 1][k][h + 1], sum[q & 1][k][h + 2], sum[q & 1][k][h + 3]};
                    else v = more[((q - 2) * NV + k) * (V / 4) * T + h / 4 * T + threadIdx.x];
                } else {
                    v = f32x4{sum[q][k][h], sum[q][k][h + 1], sum[q][k][h + 2], sum[q][k][h + 3]};
                }
                const float four[4] = {v[0], v[1], v[2], v[3]};
                if constexpr (PER == 1) elem_store<ElemF32, 4>(out, (k * G + t) * V + h, four, in[k] - h < 4 ? in[k] - h : 4);
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) cols[((threadIdx.x / G) * NV + k) * G * V + t * V + h + j] = four[j];
            }
        if constexpr (PER > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.d; c += 256) {
                float v = 0.f;
                for (int g = 0; g < PER; ++g) v += cols[g * NV * G * V + c];
                out[c] = v;
            }
        }
    }
}

struct ColArgs {
    const float* part;
    int blocks, sets, d;
    void* out[SETS];
    int type[SETS];
};

// 64 columns of one set: 16 slices of the partial rows each, then the slices.
__global__ __launch_bounds__(1024) void column_sum_kernel(ColArgs a) {
    __shared__ float sums[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6, q = blockIdx.y;
    float v = 0.f;
    if (c < a.d)
#pragma unroll 8
        for (int b = slice; b < a.blocks; b += 16) v += a.part[((int64_t)b * a.sets + q) * a.d + c];
    sums[slice][threadIdx.x & 63] = v;
    __syncthreads();
    if (slice || c >= a.d) return;
    for (int k = 1; k < 16; ++k) v += sums[k][threadIdx.x & 63];
    if (a.type[q] == GCP_TYPE_F32) ((float*)a.out[q])[c] = v;
    else if (a.type[q] == GCP_TYPE_BF16) ((__bf16*)a.out[q])[c] = (__bf16)v;
    else ((_Float16*)a.out[q])[c] = (_Float16)v;
}

// Group size and vectors per thread for a row of d elements: the smallest group that holds the row in one vector per thread, up to 256
// threads, then two vectors (16384 x 4096 bf16, an element-wise gate, both forms in one run of an earlier state: forward 135 us with 256 threads
// of two vectors against 167 with 512 of one, backward 271 against 325).
template <class E, class F>
bool by_shape(int d, F f) {
    constexpr int V = E::vec;
#define TRY(G, NV) if (d <= G * NV * V) { f(std::integral_constant<int, G>(), std::integral_constant<int, NV>()); return true; }
    TRY(8, 1) TRY(16, 1) TRY(32, 1) TRY(64, 1) TRY(128, 1) TRY(256, 1) TRY(256, 2) TRY(512, 2) TRY(1024, 2)
    if constexpr (V == 4) { TRY(1024, 4) }
#undef TRY
    return false;
}
// Workgroups of the backward: as many as the registers let reside on 256 CUs, each walking many rows, but four turns before there are more of
// them than CUs (the partial sums of each have to be added).
template <class E, int G, int NV>
int64_t backward_blocks(int64_t rows) {
    constexpr int T = G > 256 ? G : 256, most = 256 * backward_groups<E, G, NV>();
    const int64_t blocks = (rows + T / G - 1) / (T / G), few = blocks < 256 ? blocks : blocks < 1024 ? 256 : blocks / 4;
    return few < most ? few : most;
}

template <class F>
int by_type(int type, F f) {
    if (type == GCP_TYPE_F32) return f(ElemF32());
    if (type == GCP_TYPE_BF16) return f(ElemBf16());
    return f(ElemF16());
}

int check_desc(const gcp_block_norm_t* n) {
    if (!n || n->rows < 0 || n->d < 1 || !elem_type_ok(n->type) || n->post < 0 || n->post > 2 || n->pre < 0 || n->pre > 2) return GCPNET_E_BADARG;
    if (n->act < 0 || n->act > GCP_ACT_SIGMOID) return GCPNET_E_BADARG;
    if (n->param_type != GCP_TYPE_F32 && n->param_type != n->type) return GCPNET_E_BADARG;
    if (n->rows > 0 && (n->post || n->gate) && !n->y) return GCPNET_E_BADARG;
    if (n->x_ld < 0 || n->y_ld < 0 || n->gate_ld < 0) return GCPNET_E_BADARG;
    if (n->d > MAX_D || n->rows > INT32_MAX) return GCPNET_E_UNSUPPORTED;
    return 0;
}

NormArgs fill(const gcp_block_norm_t* n) {
    NormArgs a = {};
    a.rows = n->rows; a.d = n->d;
    a.x = n->x; a.y = n->y; a.gate = n->gate;
    a.x_ld = n->x_ld; a.y_ld = n->y_ld; a.gate_ld = n->gate_ld;
    a.post_w = n->post ? n->post_w : nullptr; a.post_b = n->post ? n->post_b : nullptr;
    a.pre_w = n->pre ? n->pre_w : nullptr; a.pre_b = n->pre ? n->pre_b : nullptr;
    a.post = n->post; a.pre = n->pre; a.act = n->act; a.w_f32 = n->param_type == GCP_TYPE_F32;
    a.scale = n->scale; a.slope = n->slope; a.eps = n->eps; a.inv_d = 1.f / (float)n->d;
    return a;
}

}  // namespace

int gcp_column_sums(const float* part, int blocks, int sets, int d, void* const* out, const int* type, hipStream_t stream) {
    ColArgs c = {};
    c.part = part; c.blocks = blocks; c.sets = sets; c.d = d;
    for (int q = 0; q < sets; ++q) {
        c.out[q] = out[q];
        c.type[q] = type[q];
    }
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)gcp_cdiv(d, 64), (unsigned)sets), dim3(1024), 0, stream, c);
    GCP_HIP_CHECK_LAUNCH();
    return 0;
}

extern "C" int gcpnet_block_norm_forward(const gcp_block_norm_t* n, void* s, void* h, float* stats, void* stream) {
    if (int rc = check_desc(n)) return rc;
    if (n->rows == 0) return 0;
    if (!n->x || (n->pre && !h) || !aligned16(stats)) return GCPNET_E_BADARG;
    NormArgs a = fill(n);
    a.s = s; a.h = h; a.stats = stats;
    const int piece = 16 / elem_bytes(n->type);
    auto whole = [&](const void* p, int64_t ld) { return !p || (aligned16(p) && ld % piece == 0); };
    a.once = whole(n->x, n->x_ld) && whole(n->y, n->y_ld) && whole(n->gate, n->gate_ld);
    a.once_x = a.once && n->x_ld; a.once_y = a.once && n->y_ld;  // (a row for all of them is read again)
    return by_type(n->type, [&](auto e) {
        typedef decltype(e) E;
        bool fits = true;  // (a launch has less than 2^32 threads)
        const bool ok = by_shape<E>(n->d, [&](auto g, auto nv) {
            constexpr int G = g.value, T = G > 256 ? G : 256;
            const int64_t blocks = (n->rows + T / G - 1) / (T / G);
            fits = blocks * T <= UINT32_MAX;
            if (!fits) return;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_kernel<E, G, nv.value>), dim3((unsigned)blocks), dim3(T), 0, (hipStream_t)stream, a);
        });
        if (!ok || !fits) return GCPNET_E_UNSUPPORTED;
        GCP_HIP_CHECK_LAUNCH();
        return 0;
    });
}

extern "C" int64_t gcpnet_block_norm_backward_scratch(const gcp_block_norm_t* n) {
    if (int rc = check_desc(n)) return rc;
    int64_t blocks = 0;
    by_type(n->type, [&](auto e) {
        typedef decltype(e) E;
        by_shape<E>(n->d, [&](auto g, auto nv) { blocks = backward_blocks<E, g.value, nv.value>(n->rows); });
        return 0;
    });
    return blocks * SETS * n->d;
}

extern "C" int gcpnet_block_norm_backward(const gcp_block_norm_t* n, const float* stats, const void* ds, const void* dh,
                                          void* dx, void* dy, void* dgate, void* d_post_w, void* d_post_b, void* d_pre_w, void* d_pre_b,
                                          float* scratch, void* stream) {
    if (int rc = check_desc(n)) return rc;
    if ((n->post || n->pre) && n->rows > 0 && (!stats || !aligned16(stats))) return GCPNET_E_BADARG;
    if (n->rows > 0 && n->pre && dh && !n->x) return GCPNET_E_BADARG;
    NormArgs a = fill(n);
    const bool channel = n->gate && n->gate_ld == 0;
    void* const out[SETS] = {n->pre ? d_pre_w : nullptr, n->post ? d_post_w : nullptr, n->pre ? d_pre_b : nullptr, n->post ? d_post_b : nullptr,
                             channel ? dgate : nullptr};
    void* sums[SETS];
    int types[SETS];
    for (int q = 0; q < SETS; ++q) {
        a.slot[q] = out[q] ? a.sets : -1;
        if (!out[q]) continue;
        sums[a.sets] = out[q];
        types[a.sets++] = q == 4 ? n->type : n->param_type;
    }
    if (a.sets && n->rows > 0 && !scratch) return GCPNET_E_BADARG;
    int64_t blocks = 0;
    if (n->rows > 0) {
        a.pre = n->pre && dh ? n->pre : 0;
        a.dh = n->pre ? dh : nullptr;
        a.ds = ds; a.dx = dx; a.dy = dy; a.dgate = dgate;
        a.stats = const_cast<float*>(stats);
        a.part = scratch;
        const bool bias = out[2] || out[3] || out[4];
        const int rc = by_type(n->type, [&](auto e) {
            typedef decltype(e) E;
            const bool ok = by_shape<E>(n->d, [&](auto g, auto nv) {
                constexpr int G = g.value, T = G > 256 ? G : 256;
                constexpr int NV = nv.value;
                blocks = backward_blocks<E, G, NV>(n->rows);
                // Parameters in LDS where the workgroups that should reside still do: a load of them in every turn would also wait for the row
                // requested ahead (16384 x 4096 bf16, RMS norms: 295 us against 281; layer norms 287 against 260).
                const int lds = 3 * NV * G * 16 * (E::code != GCP_TYPE_F32 && a.w_f32 ? E::vec / 4 : 1);
                const int own = backward_lds<E, G, NV>(bias);
                a.held = (a.post_w || a.post_b || a.pre_w) && lds <= 49152 && (own + lds) * backward_groups<E, G, NV>() <= 160 * 1024;
                const int dynamic = a.held ? lds : 0;
                if (bias) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<E, G, NV, true>), dim3((unsigned)blocks), dim3(T), dynamic, (hipStream_t)stream, a);
                else hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<E, G, NV, false>), dim3((unsigned)blocks), dim3(T), dynamic, (hipStream_t)stream, a);
            });
            if (!ok) return GCPNET_E_UNSUPPORTED;
            GCP_HIP_CHECK_LAUNCH();
            return 0;
        });
        if (rc) return rc;
    }
    if (a.sets) return gcp_column_sums(scratch, (int)blocks, a.sets, n->d, sums, types, (hipStream_t)stream);  // (no rows: the sums are 0)
    return 0;
}
