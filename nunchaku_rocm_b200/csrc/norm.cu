// Layer norm with a weight and a bias, forward and backward, one pass over HBM each.
//
//   y  = xh (w + add) + b         xh = (x - mean) rstd
//   dx = rstd (v - mean(v) - xh mean(v xh)),   v = dy (w + add)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row is held in registers by a team of one or more warps, so the mean is subtracted before the squares are summed (no
// cancellation) and nothing is read twice.  A team walks over many rows and keeps its columns' weights in registers, and in
// the backward pass the fp32 sums of its columns' weight gradients too: the rows of a sum are added in a fixed order, the
// teams of a CTA and then the CTAs' sums (a second small kernel) likewise, with no atomics, so two calls give the same bits.
// The next row's loads are issued before the current row is reduced.
//
// Bound: HBM.  Forward reads x and writes y, backward reads x and dy and writes dx; the partial sums are
// 8 dim bytes per CTA.
#include "nb_common.cuh"

namespace nb {
namespace {

constexpr int kMaxThreads = 512;

struct LnParams {
    const void* x; const void* w; const void* b; void* y;
    float* mean; float* rstd;
    const void* dy; void* dx;
    float* part;  // (groups, gridDim.x, 2, dim)
    long long stride_x, stride_dy, stride_w;
    int rows, dim;
    float eps, add;
};

template <typename T> __device__ __forceinline__ float ld1(const T* p) { return to_f32<T>(*p); }
template <> __device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ void st1(T* p, float v) { *p = from_f32<T>(v); }
template <> __device__ __forceinline__ void st1<float>(float* p, float v) { *p = v; }

// Eight values of a row as they are held between load and use.
template <typename T>
struct Raw {
    uint4 r;
    __device__ __forceinline__ void load(const T* p) { r = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        float2 f;
        f = unpack2<T>(r.x); v[0] = f.x; v[1] = f.y;
        f = unpack2<T>(r.y); v[2] = f.x; v[3] = f.y;
        f = unpack2<T>(r.z); v[4] = f.x; v[5] = f.y;
        f = unpack2<T>(r.w); v[6] = f.x; v[7] = f.y;
    }
    __device__ static __forceinline__ void store(T* p, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
};
template <>
struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ static __forceinline__ void store(float* p, const float (&v)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
};

// The columns of one thread: U groups of eight.  VEC: eight neighbours, 16-byte accesses.  Otherwise one value at a time,
// neighbouring threads on neighbouring columns: any dim and alignment.
template <bool VEC>
__device__ __forceinline__ int col(int u, int j, int t, int team) {
    return VEC ? (u * team + t) * 8 + j : (u * 8 + j) * team + t;
}
template <typename T, bool VEC>
struct Held {  // one group of a row
    Raw<T> raw;
    __device__ __forceinline__ void load(const T* row, int u, int t, int team, int) { raw.load(row + col<true>(u, 0, t, team)); }
    __device__ __forceinline__ void widen(float (&v)[8]) const { raw.widen(v); }
};
template <typename T>
struct Held<T, false> {
    T e[8];
    __device__ __forceinline__ void load(const T* row, int u, int t, int team, int dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col<false>(u, j, t, team);
            e[j] = c < dim ? row[c] : T(0.f);
        }
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = ld1<T>(&e[j]);
    }
};
template <typename T, bool VEC>
__device__ __forceinline__ void put(T* row, const float (&v)[8], int u, int t, int team, int dim) {
    if constexpr (VEC) {
        Raw<T>::store(row + col<true>(u, 0, t, team), v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col<false>(u, j, t, team);
            if (c < dim) st1<T>(row + c, v[j]);
        }
    }
}
template <typename W, bool VEC>
__device__ __forceinline__ void get_w(const void* base, long long off, float (&v)[8], int u, int t, int team, int dim, float none) {
    const W* row = static_cast<const W*>(base);
    if (!row) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = none;
        return;
    }
    Held<W, VEC> h;
    h.load(row + off, u, t, team, dim);
    h.widen(v);
}

// Sums of N values over a team of `warps` warps; the result is in every thread.  One warp needs no barrier; otherwise the
// CTA is one team and `red` alternates between two halves, so that one barrier per reduction is enough.
template <int N>
__device__ __forceinline__ void team_sum(float (&s)[N], int warps, float* red, int& flip) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    if (warps == 1) return;
    float* r = red + flip * (2 * kMaxThreads / 32);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) r[(threadIdx.x >> 5) * 2 + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += r[w * 2 + i];
}

// blockDim = (team, teams of a CTA); more than one team only when a team is one warp.  grid = (CTAs of a group, groups).
template <typename T, typename W, int U, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_kernel(const LnParams p) {
    __shared__ float red[4 * kMaxThreads / 32];
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5;
    const int step = gridDim.x * blockDim.y;
    const long long first = (long long)blockIdx.y * p.rows;
    int row = blockIdx.x * blockDim.y + threadIdx.y, flip = 0;
    if (row >= p.rows) return;  // a whole team
    float w[U][8], b[U][8];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        on[u] = col<VEC>(u, 0, t, team) < p.dim;
        if (!on[u]) continue;
        get_w<W, VEC>(p.w, blockIdx.y * p.stride_w, w[u], u, t, team, p.dim, 1.f);
        get_w<W, VEC>(p.b, blockIdx.y * p.stride_w, b[u], u, t, team, p.dim, 0.f);
        if (p.w)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[u][j] += p.add;
    }
    const T* x = static_cast<const T*>(p.x);
    Held<T, VEC> next[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (on[u]) next[u].load(x + (first + row) * p.stride_x, u, t, team, p.dim);
    const float inv = 1.f / (float)p.dim;
    for (; row < p.rows; row += step) {
        float v[U][8], s[1] = {0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            next[u].widen(v[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[0] += v[u][j];
        }
        if (row + step < p.rows) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (on[u]) next[u].load(x + (first + row + step) * p.stride_x, u, t, team, p.dim);
        }
        team_sum<1>(s, warps, red, flip);
        const float mean = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = VEC || col<VEC>(u, j, t, team) < p.dim ? v[u][j] - mean : 0.f;
                v[u][j] = d;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        team_sum<1>(s, warps, red, flip);
        const float rstd = rsqrtf(s[0] * inv + p.eps);
        if (t == 0 && p.mean) p.mean[first + row] = mean;
        if (t == 0 && p.rstd) p.rstd[first + row] = rstd;
        if (!p.y) continue;
        T* y = static_cast<T*>(p.y) + (first + row) * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] = fmaf(v[u][j] * rstd, w[u][j], b[u][j]);
            put<T, VEC>(y, v[u], u, t, team, p.dim);
        }
    }
}

template <typename T, typename W, int U, bool VEC, bool SUMS>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_backward_kernel(const LnParams p) {
    __shared__ float red[4 * kMaxThreads / 32];
    extern __shared__ __align__(16) float joined[];  // teams > 1: [teams][2][dim]
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5;
    const int step = gridDim.x * blockDim.y;
    const long long first = (long long)blockIdx.y * p.rows;
    int row = blockIdx.x * blockDim.y + threadIdx.y, flip = 0;
    float w[U][8], dw[U][8], db[U][8];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        on[u] = col<VEC>(u, 0, t, team) < p.dim;
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[u][j] = db[u][j] = 0.f;
        if (!on[u]) continue;
        get_w<W, VEC>(p.w, blockIdx.y * p.stride_w, w[u], u, t, team, p.dim, 1.f);
        if (p.w)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[u][j] += p.add;
    }
    const T* x = static_cast<const T*>(p.x);
    const T* dy = static_cast<const T*>(p.dy);
    Held<T, VEC> nx[U], ng[U];
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            nx[u].load(x + (first + r) * p.stride_x, u, t, team, p.dim);
            ng[u].load(dy + (first + r) * p.stride_dy, u, t, team, p.dim);
        }
        nm = p.mean[first + r];
        nr = p.rstd[first + r];
    };
    if (row < p.rows) fetch(row);
    const float inv = 1.f / (float)p.dim;
    for (; row < p.rows; row += step) {
        float xh[U][8], g[U][8], s[2] = {0.f, 0.f};
        const float mean = nm, rstd = nr;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            nx[u].widen(xh[u]);
            ng[u].widen(g[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xh[u][j] = (xh[u][j] - mean) * rstd;  // (columns behind dim: g is 0 there, and nothing is stored)
                if constexpr (SUMS) {
                    dw[u][j] = fmaf(g[u][j], xh[u][j], dw[u][j]);
                    db[u][j] += g[u][j];
                }
                g[u][j] *= w[u][j];
                s[0] += g[u][j];
                s[1] = fmaf(g[u][j], xh[u][j], s[1]);
            }
        }
        if (row + step < p.rows) fetch(row + step);
        if (!p.dx) continue;
        team_sum<2>(s, warps, red, flip);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T* dx = static_cast<T*>(p.dx) + (first + row) * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[u][j] = rstd * (g[u][j] - m0 - xh[u][j] * m1);
            put<T, VEC>(dx, g[u], u, t, team, p.dim);
        }
    }
    if constexpr (SUMS) {
        float* part = p.part + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.dim;
        if (blockDim.y == 1) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!on[u]) continue;
                put<float, VEC>(part, dw[u], u, t, team, p.dim);
                put<float, VEC>(part + p.dim, db[u], u, t, team, p.dim);
            }
        } else {
            float* mine = joined + (size_t)threadIdx.y * 2 * p.dim;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!on[u]) continue;
                put<float, VEC>(mine, dw[u], u, t, team, p.dim);
                put<float, VEC>(mine + p.dim, db[u], u, t, team, p.dim);
            }
            __syncthreads();
            for (int c = threadIdx.y * blockDim.x + t; c < 2 * p.dim; c += blockDim.x * blockDim.y) {
                float s = 0.f;
                for (int y = 0; y < (int)blockDim.y; ++y) s += joined[(size_t)y * 2 * p.dim + c];
                part[c] = s;
            }
        }
    }
}

// Sums of the CTAs' partial rows: a CTA takes 32 columns, its eight warps every eighth partial row.
template <typename W>
__global__ void __launch_bounds__(256) layer_norm_sums_kernel(const float* part, int parts, int dim, W* dw, W* db) {
    __shared__ float sum[8][32];
    const int c = blockIdx.x * 32 + threadIdx.x;  // of 2 dim: first the weight's, then the bias'
    const float* p = part + (long long)blockIdx.y * parts * 2 * dim;
    float s = 0.f;
    if (c < 2 * dim)
        for (int i = threadIdx.y; i < parts; i += 8) s += p[(long long)i * 2 * dim + c];
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < 2 * dim) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += sum[i][threadIdx.x];
        W* out = c < dim ? dw : db;
        if (out) st1<W>(out + (long long)blockIdx.y * dim + (c < dim ? c : c - dim), s);
    }
}

// How a call is laid out: threads of a team, teams of a CTA, groups of eight columns per thread, CTAs per group of rows.
struct Shape {
    int team, teams, u, ctas;
};
Shape shape_of(int groups, int rows, int dim, bool backward) {
    Shape s;
    const int eights = (dim + 7) / 8;
    s.u = eights <= 512 ? 1 : eights <= 1024 ? 2 : 4;
    if (dim <= 512) {  // a warp per row: no barriers
        s.u = eights <= 32 ? 1 : 2;
        s.team = 32;
        s.teams = 8;
    } else {
        s.team = ((eights + s.u - 1) / s.u + 31) / 32 * 32;
        s.teams = 1;
    }
    int sms = nb_num_sms();
    if (sms <= 0) sms = 148;
    const int threads = s.team * s.teams;
    // CTAs that are resident together at the kernels' register counts (about 64 and 128 per thread)
    const int resident = sms * ((backward ? 768 : 1024) / threads < 1 ? 1 : (backward ? 768 : 1024) / threads);
    const int want = (rows + s.teams - 1) / s.teams;
    int per = resident / groups;
    if (per < 1) per = 1;
    s.ctas = want < per ? want : per;
    return s;
}

template <typename T, typename W, int U, bool VEC>
int launch(const LnParams& p, const Shape& s, int groups, bool backward, cudaStream_t st) {
    const dim3 grid(s.ctas, groups), block(s.team, s.teams);
    if (!backward) {
        layer_norm_kernel<T, W, U, VEC><<<grid, block, 0, st>>>(p);
    } else {
        const size_t smem = p.part && s.teams > 1 ? (size_t)s.teams * 2 * p.dim * 4 : 0;  // at most 8 x 2 x 512 x 4 = 32 KB
        if (p.part) layer_norm_backward_kernel<T, W, U, VEC, true><<<grid, block, smem, st>>>(p);
        else layer_norm_backward_kernel<T, W, U, VEC, false><<<grid, block, 0, st>>>(p);
    }
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
template <typename T, typename W>
int launch(const LnParams& p, const Shape& s, int groups, bool vec, bool backward, cudaStream_t st) {
    switch (s.u) {
        case 1: return vec ? launch<T, W, 1, true>(p, s, groups, backward, st) : launch<T, W, 1, false>(p, s, groups, backward, st);
        case 2: return vec ? launch<T, W, 2, true>(p, s, groups, backward, st) : launch<T, W, 2, false>(p, s, groups, backward, st);
        default: return vec ? launch<T, W, 4, true>(p, s, groups, backward, st) : launch<T, W, 4, false>(p, s, groups, backward, st);
    }
}
int launch(const LnParams& p, const Shape& s, const nb_layer_norm_args* a, bool vec, bool backward, cudaStream_t st) {
    if (a->dtype == NB_DTYPE_FP32) return launch<float, float>(p, s, a->groups, vec, backward, st);
    if (a->dtype == NB_DTYPE_BF16)
        return a->w_fp32 ? launch<__nv_bfloat16, float>(p, s, a->groups, vec, backward, st)
                         : launch<__nv_bfloat16, __nv_bfloat16>(p, s, a->groups, vec, backward, st);
    return a->w_fp32 ? launch<__half, float>(p, s, a->groups, vec, backward, st) : launch<__half, __half>(p, s, a->groups, vec, backward, st);
}

int check(const nb_layer_norm_args* a) {
    NB_REQUIRE(a && a->groups > 0 && a->rows >= 0 && a->dim > 0);
    NB_REQUIRE(a->dtype == NB_DTYPE_BF16 || a->dtype == NB_DTYPE_FP16 || a->dtype == NB_DTYPE_FP32);
    if (a->dim > NB_LAYER_NORM_MAX_DIM) return fail_with(NB_ERR_UNSUPPORTED, "dim above NB_LAYER_NORM_MAX_DIM");
    if (a->groups > 65535) return fail_with(NB_ERR_TOO_LARGE, "more than 65535 groups");
    if (a->rows > (1 << 30)) return fail_with(NB_ERR_TOO_LARGE, "more than 2^30 rows in a group");
    return NB_OK;
}
LnParams params_of(const nb_layer_norm_args* a) {
    LnParams p = {};
    p.x = a->x; p.w = a->w; p.b = a->b; p.y = a->y;
    p.mean = a->mean; p.rstd = a->rstd;
    p.dy = a->dy; p.dx = a->dx;
    p.stride_x = a->stride_x; p.stride_dy = a->stride_dy; p.stride_w = a->stride_w;
    p.rows = a->rows; p.dim = a->dim; p.eps = a->eps; p.add = a->weight_add;
    return p;
}
bool vec_w(const nb_layer_norm_args* a, const void* w) {
    return !w || (aligned16(w) && (a->groups == 1 || a->stride_w % 8 == 0));
}

}  // namespace
}  // namespace nb

extern "C" int64_t nb_layer_norm_workspace_bytes(int32_t groups, int32_t rows, int32_t dim, int32_t dtype) {
    (void)dtype;
    if (groups <= 0 || rows <= 0 || dim <= 0 || dim > NB_LAYER_NORM_MAX_DIM) return 0;
    return (int64_t)nb::shape_of(groups, rows, dim, true).ctas * groups * 2 * dim * 4;
}

extern "C" int nb_layer_norm(const nb_layer_norm_args* a, void* stream) {
    using namespace nb;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return NB_OK;
    NB_REQUIRE(a->x);
    const bool vec = a->dim % 8 == 0 && aligned16(a->x) && aligned16(a->y) && a->stride_x % 8 == 0 && vec_w(a, a->w) && vec_w(a, a->b);
    return launch(params_of(a), shape_of(a->groups, a->rows, a->dim, false), a, vec, false, static_cast<cudaStream_t>(stream));
}

extern "C" int nb_layer_norm_backward(const nb_layer_norm_args* a, void* stream) {
    using namespace nb;
    if (int rc = check(a)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool sums = a->dw || a->db;
    if (a->rows == 0) {  // an empty sum
        const size_t bytes = (size_t)a->groups * a->dim * (a->w_fp32 || a->dtype == NB_DTYPE_FP32 ? 4 : 2);
        if (a->dw) NB_CUDA_CHECK(cudaMemsetAsync(a->dw, 0, bytes, st));
        if (a->db) NB_CUDA_CHECK(cudaMemsetAsync(a->db, 0, bytes, st));
        return NB_OK;
    }
    if (!sums && !a->dx) return NB_OK;
    NB_REQUIRE(a->x && a->dy && a->mean && a->rstd);
    const Shape s = shape_of(a->groups, a->rows, a->dim, true);
    LnParams p = params_of(a);
    if (sums) {
        NB_REQUIRE(a->workspace && aligned16(a->workspace));
        if (a->workspace_bytes < nb_layer_norm_workspace_bytes(a->groups, a->rows, a->dim, a->dtype))
            return fail_with(NB_ERR_INVALID, "workspace smaller than nb_layer_norm_workspace_bytes()");
        p.part = static_cast<float*>(a->workspace);
    }
    const bool vec = a->dim % 8 == 0 && aligned16(a->x) && aligned16(a->dy) && aligned16(a->dx) && a->stride_x % 8 == 0 &&
                     a->stride_dy % 8 == 0 && vec_w(a, a->w);
    if (int rc = launch(p, s, a, vec, true, st)) return rc;
    if (!sums) return NB_OK;
    const dim3 grid((2 * a->dim + 31) / 32, a->groups), block(32, 8);
    if (a->w_fp32 || a->dtype == NB_DTYPE_FP32)
        layer_norm_sums_kernel<float><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<float*>(a->dw), static_cast<float*>(a->db));
    else if (a->dtype == NB_DTYPE_BF16)
        layer_norm_sums_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<__nv_bfloat16*>(a->dw), static_cast<__nv_bfloat16*>(a->db));
    else
        layer_norm_sums_kernel<__half><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<__half*>(a->dw), static_cast<__half*>(a->db));
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
