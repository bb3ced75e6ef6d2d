// The norms before and after a residual block with its gate and residual scale, forward and backward:
//
//   u = post(y);  s = x + scale * act(gate) * u;  h = pre(s)              post, pre: layer norm, RMS norm or none
//
//   n2 = (s - mean2) rstd2;  gs = ds + rstd2 (dh w - mean(dh w) - n2 mean(dh w n2))      (RMS: without the mean)
//   dx = gs;  du = scale act(gate) gs;  dgate = scale gs u act'(gate);  dy = rstd1 (du w - mean(du w) - n1 mean(du w n1))
//   weights and biases: column sums of dh n2, dh, du n1, du, and of dgate for a gate of one value per channel.
//
// Bound: HBM -- forward reads x, y (and an element-wise gate) and writes s, h; backward reads y, s, ds, dh, writes dx, dy.  A row is
// held in the registers of a group of 8 to 1024 threads between its reductions, so everything is read once; the statistics take
// two passes over the registers (mean, then squares of the differences).  The backward's groups walk many rows and keep the column sums
// in registers; one partial sum per workgroup goes through memory, summed in a fixed order by a second launch.
#include <initializer_list>
#include <type_traits>

#include "elem_types.h"
#include "linear_tiles.h"

namespace {

constexpr int MAX_D = 16384, BWD_BLOCKS = 512, SETS = 5;  // sets of column sums: pre_w, pre_b, post_w, post_b, gate

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
};

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
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < G / 64; ++w) t += lds[turn][k][w];
            v[k] = t;
        }
        turn ^= 1;
    }
}

template <class E, int G, int NV, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_fwd_kernel(NormArgs a) {
    constexpr int PER = (G > 256 ? G : 256) / G;  // groups of a workgroup
    __shared__ float lds[2][2][16];
    int turn = 0;
    const int t = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
    const bool on = row < a.rows;  // (a group of 256 or more is one workgroup: its rows are all on)
    const int64_t r = on ? row : 0;
    float u[NV][V], s[NV][V];
    bool in[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) in[k] = (k * G + t) * V < a.d;
    Raw<E, V> xr[NV], yr[NV], gr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * G + t) * V;
        elem_zero<E, V>(xr[k]);
        elem_zero<E, V>(yr[k]);
        elem_zero<E, V>(gr[k]);
        if (in[k]) {
            xr[k] = elem_load<E, V>(a.x, r * a.x_ld + c);
            if (a.y) yr[k] = elem_load<E, V>(a.y, r * a.y_ld + c);
            if (a.gate) gr[k] = elem_load<E, V>(a.gate, r * a.gate_ld + c);
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) u[k][j] = (float)yr[k].x[j];
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
                z[k][j] = in[k] ? z[k][j] - mean : 0.f;
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
        const int c = (k * G + t) * V;
        if (!in[k]) {
#pragma unroll
            for (int j = 0; j < V; ++j) s[k][j] = 0.f;
            continue;
        }
        float w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
        param_load<E, V>(a.post_w, c, a.w_f32, w);
        param_load<E, V>(a.post_b, c, a.w_f32, b);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float z = u[k][j];
            if (a.post) z = fmaf(z, w[j], b[j]);
            if (a.gate) z *= gcp_act(a.act, (float)gr[k].x[j], a.slope);
            s[k][j] = a.y ? fmaf(a.scale, z, (float)xr[k].x[j]) : (float)xr[k].x[j];
        }
        if (on && a.s) elem_store<E, V>(a.s, r * a.d + c, s[k]);
    }
    if (a.pre) {
        normalize(s, a.pre, st[2], st[3]);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V;
            if (!in[k]) continue;
            float w[V], b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            param_load<E, V>(a.pre_w, c, a.w_f32, w);
            param_load<E, V>(a.pre_b, c, a.w_f32, b);
#pragma unroll
            for (int j = 0; j < V; ++j) s[k][j] = fmaf(s[k][j], w[j], b[j]);
            if (on) elem_store<E, V>(a.h, r * a.d + c, s[k]);
        }
    }
    if (a.stats && on && t == 0) *(f32x4*)(a.stats + 4 * r) = f32x4{st[0], st[1], st[2], st[3]};
}

template <class E, int G, int NV, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_bwd_kernel(NormArgs a) {
    constexpr int PER = (G > 256 ? G : 256) / G;
    __shared__ float lds[2][2][16];
    __shared__ float cols[PER > 1 ? 256 * NV * V : 1];
    int turn = 0;
    const int t = threadIdx.x % G;
    bool in[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) in[k] = (k * G + t) * V < a.d;
    float sum[SETS][NV][V];
#pragma unroll
    for (int q = 0; q < SETS; ++q)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[q][k][j] = 0.f;
    const bool channel = a.gate && a.gate_ld == 0;
    // (all groups of a workgroup make the same number of turns: barriers and shuffles stay in step)
    for (int64_t first = (int64_t)blockIdx.x * PER; first < a.rows; first += (int64_t)gridDim.x * PER) {
        const int64_t row = first + threadIdx.x / G;
        const bool on = row < a.rows;
        const int64_t r = on ? row : 0;
        Raw<E, V> yr[NV], sr[NV], gr[NV], dsr[NV], dhr[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V;
            elem_zero<E, V>(yr[k]); elem_zero<E, V>(sr[k]); elem_zero<E, V>(gr[k]); elem_zero<E, V>(dsr[k]); elem_zero<E, V>(dhr[k]);
            if (in[k] && on) {
                if (a.y) yr[k] = elem_load<E, V>(a.y, r * a.y_ld + c);
                if (a.pre) sr[k] = elem_load<E, V>(a.s, r * a.x_ld + c);
                if (a.gate) gr[k] = elem_load<E, V>(a.gate, r * a.gate_ld + c);
                if (a.ds) dsr[k] = elem_load<E, V>(a.ds, r * a.d + c);
                if (a.dh) dhr[k] = elem_load<E, V>(a.dh, r * a.d + c);
            }
        }
        f32x4 st = {0.f, 1.f, 0.f, 1.f};
        if (on && a.stats) st = *(const f32x4*)(a.stats + 4 * r);
        float gs[NV][V];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) gs[k][j] = (float)dsr[k].x[j];
        if (a.dh) {
            float m[2] = {0.f, 0.f}, dn[NV][V];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float w[V];
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = 1.f;
                if (in[k]) param_load<E, V>(a.pre_w, (k * G + t) * V, a.w_f32, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float dh = (float)dhr[k].x[j], n = ((float)sr[k].x[j] - st[2]) * st[3];
                    dn[k][j] = dh * w[j];  // (0 outside)
                    m[0] += dn[k][j];
                    m[1] += dn[k][j] * n;
                    sum[0][k][j] += dh * n;
                    sum[1][k][j] += dh;
                }
            }
            group_sum<G, 2>(m, lds, turn);
            const float m0 = a.pre == GCP_NORM_LAYER ? m[0] * a.inv_d : 0.f, m1 = m[1] * a.inv_d;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float n = ((float)sr[k].x[j] - st[2]) * st[3];
                    gs[k][j] += st[3] * (dn[k][j] - m0 - n * m1);
                }
        }
        if (a.dx)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (in[k] && on) elem_store<E, V>(a.dx, r * a.d + (k * G + t) * V, gs[k]);
        if (!a.y) continue;
        float du[NV][V], m[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * G + t) * V;
            float w[V], b[V], dg[V];
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            if (in[k]) {
                param_load<E, V>(a.post_w, c, a.w_f32, w);
                param_load<E, V>(a.post_b, c, a.w_f32, b);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float y = (float)yr[k].x[j], g = (float)gr[k].x[j], n = (y - st[0]) * st[1];
                const float u = a.post ? fmaf(n, w[j], b[j]) : y, q = in[k] && on ? a.scale * gs[k][j] : 0.f;
                du[k][j] = a.gate ? q * gcp_act(a.act, g, a.slope) : q;
                dg[j] = q * u * gcp_act_grad(a.act, g, a.slope);
                sum[4][k][j] += dg[j];
                sum[2][k][j] += du[k][j] * n;
                sum[3][k][j] += du[k][j];
                if (a.post) {
                    du[k][j] *= w[j];
                    m[0] += du[k][j];
                    m[1] += du[k][j] * n;
                }
            }
            if (a.dgate && !channel && in[k] && on) elem_store<E, V>(a.dgate, r * a.d + c, dg);
        }
        if (a.post) {
            group_sum<G, 2>(m, lds, turn);
            const float m0 = a.post == GCP_NORM_LAYER ? m[0] * a.inv_d : 0.f, m1 = m[1] * a.inv_d;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) du[k][j] = st[1] * (du[k][j] - m0 - ((float)yr[k].x[j] - st[0]) * st[1] * m1);
        }
        if (a.dy)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (in[k] && on) elem_store<E, V>(a.dy, r * a.d + (k * G + t) * V, du[k]);
    }
    // column sums: over the groups of the workgroup through LDS, then one partial row of each set that is wanted
#pragma unroll
    for (int q = 0; q < SETS; ++q) {
        if (a.slot[q] < 0) continue;  // (uniform)
        float* out = a.part + ((int64_t)blockIdx.x * a.sets + a.slot[q]) * a.d;
        if constexpr (PER == 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (in[k])
#pragma unroll
                    for (int j = 0; j < V; ++j) out[(k * G + t) * V + j] = sum[q][k][j];
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) cols[((threadIdx.x / G) * NV + k) * G * V + t * V + j] = sum[q][k][j];
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

// Group size and vectors per thread for a row of d elements: the smallest group that holds the row in one vector per thread, up to a
// wave, then more vectors, then 256 and 1024 threads.  Rows whose addresses do not allow 16-byte pieces go element by element.
template <class E, class F>
bool by_shape(int d, bool vec, F f) {
    constexpr int V = E::vec;
#define TRY(G, NV, VV) if (d <= G * NV * VV) { f(std::integral_constant<int, G>(), std::integral_constant<int, NV>(), std::integral_constant<int, VV>()); return true; }
    if (vec) {
        TRY(8, 1, V) TRY(16, 1, V) TRY(32, 1, V) TRY(64, 1, V) TRY(64, 2, V) TRY(256, 1, V) TRY(256, 2, V) TRY(1024, 1, V) TRY(1024, 2, V)
        if constexpr (V == 4) { TRY(1024, 4, V) }
    } else {
        TRY(16, 1, 1) TRY(64, 1, 1) TRY(64, 4, 1) TRY(64, 16, 1) TRY(256, 8, 1) TRY(1024, 4, 1) TRY(1024, 16, 1)
    }
#undef TRY
    return false;
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

// 16-byte pieces: every row of every operand starts at a multiple of 16 bytes and is whole pieces long
bool whole_pieces(const gcp_block_norm_t* n, std::initializer_list<const void*> more) {
    const int v = 16 / elem_bytes(n->type);
    if (n->d % v || n->x_ld % v || (n->y && n->y_ld % v) || (n->gate && n->gate_ld % v)) return false;
    for (const void* p : {n->x, n->y, n->gate}) if (!aligned16(p)) return false;
    for (const void* p : {n->post_w, n->post_b, n->pre_w, n->pre_b}) if (!aligned16(p)) return false;
    for (const void* p : more) if (!aligned16(p)) return false;
    return true;
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
    const bool vec = whole_pieces(n, {s, h, stats});
    return by_type(n->type, [&](auto e) {
        typedef decltype(e) E;
        const bool ok = by_shape<E>(n->d, vec, [&](auto g, auto nv, auto v) {
            constexpr int G = g.value, T = G > 256 ? G : 256;
            const int64_t blocks = (n->rows + T / G - 1) / (T / G);
            hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_kernel<E, G, nv.value, v.value>), dim3((unsigned)blocks), dim3(T), 0, (hipStream_t)stream, a);
        });
        if (!ok) return GCPNET_E_UNSUPPORTED;
        GCP_HIP_CHECK_LAUNCH();
        return 0;
    });
}

extern "C" int64_t gcpnet_block_norm_backward_scratch(int64_t rows, int d) {
    if (rows < 0 || d < 1) return GCPNET_E_BADARG;
    return (int64_t)(rows < BWD_BLOCKS ? rows : BWD_BLOCKS) * SETS * d;
}

extern "C" int gcpnet_block_norm_backward(const gcp_block_norm_t* n, const void* s, const float* stats, const void* ds, const void* dh,
                                          void* dx, void* dy, void* dgate, void* d_post_w, void* d_post_b, void* d_pre_w, void* d_pre_b,
                                          float* scratch, void* stream) {
    if (int rc = check_desc(n)) return rc;
    if ((n->post || n->pre) && n->rows > 0 && (!stats || !aligned16(stats))) return GCPNET_E_BADARG;
    if (n->rows > 0 && n->pre && dh && !s) return GCPNET_E_BADARG;
    NormArgs a = fill(n);
    const bool channel = n->gate && n->gate_ld == 0;
    void* const out[SETS] = {n->pre ? d_pre_w : nullptr, n->pre ? d_pre_b : nullptr, n->post ? d_post_w : nullptr, n->post ? d_post_b : nullptr,
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
        a.s = const_cast<void*>(s);
        a.pre = n->pre && dh ? n->pre : 0;
        a.dh = n->pre ? dh : nullptr;
        a.ds = ds; a.dx = dx; a.dy = dy; a.dgate = dgate;
        a.stats = const_cast<float*>(stats);
        a.part = scratch;
        const bool vec = whole_pieces(n, {s, ds, dh, dx, dy, dgate, stats});
        const int rc = by_type(n->type, [&](auto e) {
            typedef decltype(e) E;
            const bool ok = by_shape<E>(n->d, vec, [&](auto g, auto nv, auto v) {
                constexpr int G = g.value, T = G > 256 ? G : 256;
                blocks = (n->rows + T / G - 1) / (T / G);
                if (blocks > BWD_BLOCKS) blocks = BWD_BLOCKS;
                hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<E, G, nv.value, v.value>), dim3((unsigned)blocks), dim3(T), 0, (hipStream_t)stream, a);
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
