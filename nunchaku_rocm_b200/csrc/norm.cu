// Layer norm with a weight and a bias, forward and backward, one pass over HBM each.
//
//   y  = xh (w + add) + b         xh = (x - mean) rstd
//   dx = rstd (v - mean(v) - xh mean(v xh)),   v = dy (w + add)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A team of one or more warps has a row at a time; the mean is subtracted before the squares are summed (no cancellation)
// and nothing is read from HBM twice.  The mean is a sum of two fp32 values, the second what the first one's rounding left (the
// sum of the differences, which are exact where it matters): a row of one value has a variance of zero and gives the bias, and
// a mean far above the deviation costs y nothing.  The backward pass reads the mean as one fp32 value (xh is off by its half
// step times rstd, as in the plain form).  Differences are taken before anything is multiplied by rstd.
//
// A team walks over many rows and keeps its columns' weights in registers, and in the backward pass the fp32 sums of its
// columns' weight gradients too: the rows of a sum are added in a fixed order, the teams of a CTA and then the CTAs' sums (a
// second small kernel) likewise, with no atomics, so two calls give the same bits.
//
// Bound: HBM.  Forward reads x and writes y, backward reads x and dy and writes dx; the partial sums are 8 dim bytes per
// CTA.  What has to be covered is the latency of a row's load and of its reductions (shuffles, a barrier): the RING kernels
// keep several rows of every team on their way into shared memory (cp.async; a thread copies just the columns that it reads
// itself, so no barrier guards a row) and reduce RB rows together.
//
// Measured on a B200, back to back: 32761 x 5120 fp16, forward 119 us (5.6 TB/s; a copy of the tensor takes 109), backward and
// sums 223 (4.5 TB/s; a sum of two such tensors takes 146); 9216 x 3072 bf16 with a scale and shift per sample, 30.5 and 48.7 us
// (a copy 24.3, a sum 28.8); 8192 x 1001 bf16, which no 16 bytes divide, 20.7 and 39.1 us (floors 5.0 and 7.5).  The long
// backward pass runs at two CTAs per SM (registers of the column sums and the ring both allow no third): what remains are the
// waits of a row's own reductions.  Above 8192 channels (four groups of columns a thread) the column sums do not fit the
// registers: 270 to 480 bytes of a thread spill with a ring, 1530 to 1940 without one, and 4096 x 12288 bf16 takes 49.6 and 105
// us (floors 30.7 and 46.1).
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

// The columns of one thread: U groups of eight.  RING: eight neighbours, 16-byte accesses.  Otherwise one value at a time,
// neighbouring threads on neighbouring columns: any dim and alignment.
template <bool RING>
__device__ __forceinline__ int col(int u, int j, int t, int team) {
    return RING ? (u * team + t) * 8 + j : (u * 8 + j) * team + t;
}
template <typename T>
struct Held {  // one group of a row, one value at a time
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
template <typename T, bool RING>
__device__ __forceinline__ void put(T* row, const float (&v)[8], int u, int t, int team, int dim) {
    if constexpr (RING) {
        Raw<T>::store(row + col<true>(u, 0, t, team), v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col<false>(u, j, t, team);
            if (c < dim) st1<T>(row + c, v[j]);
        }
    }
}
template <typename W, bool RING>
__device__ __forceinline__ void get_w(const void* base, long long off, float (&v)[8], int u, int t, int team, int dim, float none) {
    const W* row = static_cast<const W*>(base);
    if (!row) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = none;
    } else if constexpr (RING) {
        Raw<W> r;
        r.load(row + off + col<true>(u, 0, t, team));
        r.widen(v);
    } else {
        Held<W> h;
        h.load(row + off, u, t, team, dim);
        h.widen(v);
    }
}

// Sums of N values over a team of `warps` warps; the result is in every thread.  One warp needs no barrier; otherwise the
// CTA is one team and `red` alternates between two halves, so that one barrier per reduction is enough.
constexpr int kRed = 2 * 2 * kMaxThreads / 32;  // two halves of two values per warp
template <int N>
__device__ __forceinline__ void team_sum(float (&s)[N], int warps, int t, float* red, int& flip) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    if (warps == 1) return;
    float* r = red + flip * (kRed / 2);
    flip ^= 1;
    if ((t & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) r[(t >> 5) * N + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += r[w * N + i];
}

// 1 / sqrt(var + eps) from the sums of the squares and of the values about a point that the mean is `rest` away from.
__device__ __forceinline__ float rstd_of(float squares, float sum, float rest, float per_row, float eps) {
    const float var = fmaf(-sum, rest, squares) * per_row, v = (var < 0.f ? 0.f : var) + eps;
    const float r = rsqrtf(v), e = fmaf(-v * r, r, 1.f);  // one step of Newton's method: rsqrtf's last bits showed
    return isfinite(e) ? fmaf(0.5f * e, r, r) : r;
}
// `sum` / n, exact where it is a value of fp32; `per` is 1 / n rounded.
__device__ __forceinline__ float quotient(float sum, float n, float per) {
    const float q = sum * per;
    return fmaf(fmaf(-q, n, sum), per, q);
}

// blockDim = (team, teams of a CTA); more than one team only when a team is one warp.  grid = (CTAs of a group, groups).
template <typename T, typename W, int U>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_kernel(const LnParams p) {
    __shared__ float red[kRed];
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5;
    const int step = gridDim.x * blockDim.y;
    const long long first = (long long)blockIdx.y * p.rows;
    int row = blockIdx.x * blockDim.y + threadIdx.y, flip = 0;
    if (row >= p.rows) return;  // a whole team
    float w[U][8], b[U][8];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        on[u] = col<false>(u, 0, t, team) < p.dim;
        if (!on[u]) continue;
        get_w<W, false>(p.w, blockIdx.y * p.stride_w, w[u], u, t, team, p.dim, 1.f);
        get_w<W, false>(p.b, blockIdx.y * p.stride_w, b[u], u, t, team, p.dim, 0.f);
        if (p.w)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[u][j] += p.add;
    }
    const T* x = static_cast<const T*>(p.x);
    Held<T> next[U];
    const float inv = 1.f / (float)p.dim;
    float next0 = ld1<T>(x + (first + row) * p.stride_x);  // a row's first value, which the others' differences are taken from
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (on[u]) next[u].load(x + (first + row) * p.stride_x, u, t, team, p.dim);
    for (; row < p.rows; row += step) {
        float v[U][8], s[1] = {0.f};
        const float x0 = next0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            next[u].widen(v[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[0] += col<false>(u, j, t, team) < p.dim ? v[u][j] - x0 : 0.f;
        }
        if (row + step < p.rows) {
            next0 = ld1<T>(x + (first + row + step) * p.stride_x);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (on[u]) next[u].load(x + (first + row + step) * p.stride_x, u, t, team, p.dim);
        }
        team_sum<1>(s, warps, t, red, flip);
        const float mean = fmaf(s[0], inv, x0);
        float d2[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = col<false>(u, j, t, team) < p.dim ? v[u][j] - mean : 0.f;
                v[u][j] = d;
                d2[0] += d;
                d2[1] = fmaf(d, d, d2[1]);
            }
        }
        team_sum<2>(d2, warps, t, red, flip);
        const float rest = d2[0] * inv, rstd = rstd_of(d2[1], d2[0], rest, inv, p.eps);  // what the mean lacks
        if (t == 0 && p.mean) p.mean[first + row] = mean + rest;
        if (t == 0 && p.rstd) p.rstd[first + row] = rstd;
        if (!p.y) continue;
        T* y = static_cast<T*>(p.y) + (first + row) * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] = fmaf((v[u][j] - rest) * rstd, w[u][j], b[u][j]);
            put<T, false>(y, v[u], u, t, team, p.dim);
        }
    }
}

// The CTA's sums of the weight's and bias' gradients into its partial row, its teams' in order.
template <int U, bool RING>
__device__ __forceinline__ void leave_sums(const LnParams& p, const float (&dw)[U][8], const float (&db)[U][8], const bool (&on)[U], float* joined) {
    const int t = threadIdx.x, team = blockDim.x;
    float* part = p.part + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.dim;
    if (blockDim.y == 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            put<float, RING>(part, dw[u], u, t, team, p.dim);
            put<float, RING>(part + p.dim, db[u], u, t, team, p.dim);
        }
    } else {
        float* mine = joined + (size_t)threadIdx.y * 2 * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
            put<float, RING>(mine, dw[u], u, t, team, p.dim);
            put<float, RING>(mine + p.dim, db[u], u, t, team, p.dim);
        }
        __syncthreads();
        for (int c = threadIdx.y * blockDim.x + t; c < 2 * p.dim; c += blockDim.x * blockDim.y) {
            float s = 0.f;
            for (int y = 0; y < (int)blockDim.y; ++y) s += joined[(size_t)y * 2 * p.dim + c];
            part[c] = s;
        }
    }
}

template <typename T, typename W, int U, bool SUMS>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_backward_kernel(const LnParams p) {
    __shared__ float red[kRed];
    extern __shared__ __align__(16) float joined[];  // teams > 1: [teams][2][dim]
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5;
    const int step = gridDim.x * blockDim.y;
    const long long first = (long long)blockIdx.y * p.rows;
    int row = blockIdx.x * blockDim.y + threadIdx.y, flip = 0;
    float w[U][8], dw[U][8], db[U][8];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        on[u] = col<false>(u, 0, t, team) < p.dim;
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[u][j] = db[u][j] = 0.f;
        if (!on[u]) continue;
        get_w<W, false>(p.w, blockIdx.y * p.stride_w, w[u], u, t, team, p.dim, 1.f);
        if (p.w)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[u][j] += p.add;
    }
    const T* x = static_cast<const T*>(p.x);
    const T* dy = static_cast<const T*>(p.dy);
    Held<T> nx[U], ng[U];
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
                xh[u][j] = col<false>(u, j, t, team) < p.dim ? (xh[u][j] - mean) * rstd : 0.f;  // (g is 0 there too)
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
        team_sum<2>(s, warps, t, red, flip);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T* dx = static_cast<T*>(p.dx) + (first + row) * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!on[u]) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[u][j] = rstd * (g[u][j] - m0 - xh[u][j] * m1);
            put<T, false>(dx, g[u], u, t, team, p.dim);
        }
    }
    if constexpr (SUMS) leave_sums<U, false>(p, dw, db, on, joined);
}

// Eight values as four pairs: the packed fp32 instructions do two at a time.
struct Eight {
    uint64_t v[4];
};
template <typename T>
__device__ __forceinline__ Eight widen_pairs(const uint4& a, const uint4& b) {
    Eight e;
    if constexpr (sizeof(T) == 4) {
        e.v[0] = pack_u32x2(a.x, a.y); e.v[1] = pack_u32x2(a.z, a.w); e.v[2] = pack_u32x2(b.x, b.y); e.v[3] = pack_u32x2(b.z, b.w);
    } else {
        const float2 f0 = unpack2<T>(a.x), f1 = unpack2<T>(a.y), f2 = unpack2<T>(a.z), f3 = unpack2<T>(a.w);
        e.v[0] = pack_f32x2(f0.x, f0.y); e.v[1] = pack_f32x2(f1.x, f1.y); e.v[2] = pack_f32x2(f2.x, f2.y); e.v[3] = pack_f32x2(f3.x, f3.y);
    }
    return e;
}
__device__ __forceinline__ uint64_t both(float x) { return pack_f32x2(x, x); }
__device__ __forceinline__ float sum_pairs(uint64_t a) {
    const float2 f = unpack_f32x2(a);
    return f.x + f.y;
}
template <typename T>
__device__ __forceinline__ void put_pairs(T* at, const Eight& e) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_f32x2(e.v[k]);
        v[2 * k] = f.x; v[2 * k + 1] = f.y;
    }
    Raw<T>::store(at, v);
}
template <typename W>
__device__ __forceinline__ Eight get_pairs(const void* base, long long off, int c, float none, float add) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = none;
    if (base) {
        Raw<W> r;
        r.load(static_cast<const W*>(base) + off + c);
        r.widen(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += add;
    }
    Eight e;
#pragma unroll
    for (int k = 0; k < 4; ++k) e.v[k] = pack_f32x2(v[2 * k], v[2 * k + 1]);
    return e;
}

// Sums of N (1, 2 or 4) values over a warp: N - 1 exchanges leave each lane one value to add up, so that four values take
// six shuffles instead of twenty.  Value k's sum comes back in the lanes from 32 k / N on.
template <int N>
__device__ __forceinline__ float warp_sums(const float (&s)[N]) {
    const int lane = threadIdx.x & 31;
    float a;
    if constexpr (N == 4) {
        const bool up = lane & 16;
        float k0 = up ? s[2] : s[0], k1 = up ? s[3] : s[1];
        k0 += __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
        k1 += __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
        const bool up2 = lane & 8;
        a = (up2 ? k1 : k0) + __shfl_xor_sync(0xffffffffu, up2 ? k0 : k1, 8);
    } else if constexpr (N == 2) {
        const bool up = lane & 16;
        a = (up ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, up ? s[0] : s[1], 16);
        a += __shfl_xor_sync(0xffffffffu, a, 8);
    } else {
        a = s[0] + __shfl_xor_sync(0xffffffffu, s[0], 16);
        a += __shfl_xor_sync(0xffffffffu, a, 8);
    }
    a += __shfl_xor_sync(0xffffffffu, a, 4);
    a += __shfl_xor_sync(0xffffffffu, a, 2);
    return a + __shfl_xor_sync(0xffffffffu, a, 1);
}

// The rows of a team in its ring: slot (i % ST) holds row i of the team's walk, x and (backward) dy one behind the other.
// Every thread copies and reads its own columns.
template <typename T, int U, int ST, bool TWO>
struct Ring {
    static constexpr int PIECES = 8 * sizeof(T) / 16;
    uint32_t base;
    int slot, half;  // bytes
    __device__ __forceinline__ Ring(unsigned char* smem, int team) {
        half = team * U * PIECES * 16;
        slot = (TWO ? 2 : 1) * half;
        base = smem_u32(smem) + threadIdx.y * ST * slot;
    }
    __device__ __forceinline__ uint32_t at(int i, int which, int u, int k, int t, int team) const {
        return base + (i % ST) * slot + which * half + ((k * U + u) * team + t) * 16;
    }
    __device__ __forceinline__ void fill(int i, int which, const T* row, bool last, int t, int team) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u == U - 1 && !last) continue;
            const T* src = row + col<true>(u, 0, t, team);
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(i, which, u, k, t, team)), "l"(src + k * 4) : "memory");
        }
    }
    __device__ __forceinline__ Eight read(int i, int which, int u, int t, int team) const {
        uint4 r[2];
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[k].x), "=r"(r[k].y), "=r"(r[k].z), "=r"(r[k].w)
                         : "r"(at(i, which, u, k, t, team)) : "memory");
        return widen_pairs<T>(r[0], r[PIECES - 1]);
    }
};
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The forward pass with a ring.  The mean and the variance take ONE round over the team without cancellation: a thread takes
// its own values' mean off before it squares, and such partial results (count n, a point near their mean, the sums r of the
// differences from it and q of their squares) are moved to a common point, `off` away, by  q += off (2 r + off n),  r += off n:
// first to the warp's mean, then to the first warp's.  RB rows go through a round together; one warp joins the warps' results
// of a row for the others.  16-bit rows have no r of their own in a thread or a warp, and the mean is one fp32 value: it is at
// most 2^11 deviations away unless all values are alike, so its rounding is 2^-14 of one (at 32761 x 5120 fp16 119 us; 129 with
// both as in fp32).
template <typename T, typename W, int U, int ST, int RB, int MT, int MB>
__global__ void __launch_bounds__(MT, MB) layer_norm_ring_kernel(const LnParams p) {
    constexpr bool REST = sizeof(T) == 4;
    __shared__ float4 red[RB][MT / 32];
    __shared__ float4 joint[RB];
    extern __shared__ __align__(16) unsigned char smem[];
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5, lane = t & 31, warp = t >> 5;
    const int step = gridDim.x * blockDim.y, row0 = blockIdx.x * blockDim.y + threadIdx.y;
    const long long first = (long long)blockIdx.y * p.rows;
    if (row0 >= p.rows) return;  // a whole team
    const Ring<T, U, ST, false> ring(smem, team);
    // all groups but the last are whole: a team of U > 1 groups has at most dim / 8 / (U - 1) threads
    const bool last = col<true>(U - 1, 0, t, team) < p.dim;
    const float count = 8.f * (U - 1) + (last ? 8.f : 0.f);
    const int mine = (p.rows - row0 + step - 1) / step;  // rows of this team
    const T* next = static_cast<const T*>(p.x) + (first + row0) * p.stride_x;
    const long long ahead = step * p.stride_x, along = (long long)step * p.dim;
    auto fill = [&](int i) {
        if (i < mine) ring.fill(i, 0, next, last, t, team);
        next += ahead;
        commit();
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) fill(i);
    T* y = static_cast<T*>(p.y) + (first + row0) * p.dim;
    Eight w[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u == U - 1 && !last) continue;
        w[u] = get_pairs<W>(p.w, blockIdx.y * p.stride_w, col<true>(u, 0, t, team), 1.f, p.add);
        b[u] = get_pairs<W>(p.b, blockIdx.y * p.stride_w, col<true>(u, 0, t, team), 0.f, 0.f);
    }
    const float own[1] = {count};
    const float in_warp = warp_sums<1>(own);
    const float per_own = count > 0.f ? 1.f / count : 0.f, per_warp = in_warp > 0.f ? 1.f / in_warp : 0.f, per_row = 1.f / (float)p.dim;
    // (what the joining lane needs of warp `lane`: its columns are the same in every row)
    float their_count = 0.f;
    for (int u = 0; u < U; ++u) {
        const int c0 = (u * team + lane * 32) * 8, c1 = c0 + 256;
        if (lane < warps) their_count += (float)(min(max(p.dim - c0, 0), c1 - c0));
    }

    for (int i = 0; i < mine; i += RB) {
        wait_but<ST - RB>();
        float mean_own[RB], pivot[RB], s[RB], q[RB], left[RB];
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            Eight d[U];
            uint64_t a = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == U - 1 && !last) continue;
                d[u] = ring.read(i + r, 0, u, t, team);
                a = add_f32x2(a, add_f32x2(add_f32x2(d[u].v[0], d[u].v[1]), add_f32x2(d[u].v[2], d[u].v[3])));
            }
            // exact for values that are all alike: 16 bits of them or a power of two have an exact sum, else differences have
            s[r] = sum_pairs(a);
            mean_own[r] = U > 2 && !REST ? quotient(s[r], count, per_own) : s[r] * per_own;
            if constexpr (U > 2 && REST) {
                const float x0 = unpack_f32x2(d[0].v[0]).x;
                const uint64_t m0 = both(-x0);
                a = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (u == U - 1 && !last) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k) a = add_f32x2(a, add_f32x2(d[u].v[k], m0));
                }
                mean_own[r] = fmaf(sum_pairs(a), per_own, x0);
            }
            if constexpr (REST) {  // (differences from the first lane's, for the warp's mean)
                pivot[r] = __shfl_sync(0xffffffffu, mean_own[r], 0);
                s[r] = count > 0.f ? (mean_own[r] - pivot[r]) * count : 0.f;
            }
            const uint64_t m = both(-mean_own[r]);
            uint64_t rest = 0;
            a = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == U - 1 && !last) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t off = add_f32x2(d[u].v[k], m);
                    a = fma_f32x2(off, off, a);
                    if constexpr (REST) rest = add_f32x2(off, rest);
                }
            }
            q[r] = sum_pairs(a);
            left[r] = sum_pairs(rest);
        }
        const float ws = warp_sums<RB>(s);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            s[r] = __shfl_sync(0xffffffffu, ws, r * (32 / RB));
            s[r] = REST ? fmaf(s[r], per_warp, pivot[r]) : quotient(s[r], in_warp, per_warp);  // the warp's mean
            const float off = count > 0.f ? mean_own[r] - s[r] : 0.f;
            q[r] = REST ? fmaf(off, fmaf(off, count, 2.f * left[r]), q[r]) : fmaf(off * off, count, q[r]);
            left[r] = fmaf(off, count, left[r]);
        }
        const float wq = warp_sums<RB>(q), wl = REST ? warp_sums<RB>(left) : 0.f;
        float mean[RB], rest[RB], rstd[RB];  // the mean is mean + rest
        if (warps == 1) {
            const float mine_rest = wl * per_row, mine_rstd = rstd_of(wq, wl, mine_rest, per_row, p.eps);  // of the row that this lane has
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                mean[r] = s[r];
                rest[r] = REST ? __shfl_sync(0xffffffffu, mine_rest, r * (32 / RB)) : 0.f;
                rstd[r] = __shfl_sync(0xffffffffu, mine_rstd, r * (32 / RB));
            }
        } else {
#pragma unroll
            for (int r = 0; r < RB; ++r)
                if (lane == r * (32 / RB)) red[r][warp] = make_float4(s[r], wq, wl, 0.f);
            __syncthreads();
            for (int r = warp; r < RB; r += warps) {
                const float4 v = lane < warps ? red[r][lane] : make_float4(0.f, 0.f, 0.f, 0.f);
                const float m = __shfl_sync(0xffffffffu, v.x, 0), off = lane < warps ? v.x - m : 0.f;
                const float both_sums[2] = {fmaf(off, fmaf(off, their_count, 2.f * v.z), v.y), fmaf(off, their_count, v.z)};
                const float sq = warp_sums<2>(both_sums), sl = __shfl_down_sync(0xffffffffu, sq, 16), c = sl * per_row;  // (lane 0)
                if (lane == 0) joint[r] = make_float4(REST ? m : m + c, c, rstd_of(sq, sl, c, per_row, p.eps), 0.f);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                const float4 v = joint[r];
                mean[r] = v.x;
                rest[r] = REST ? v.y : 0.f;
                rstd[r] = v.z;
            }
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            if (i + r >= mine) continue;  // (its slot holds an older row)
            if (t == 0 && p.mean) p.mean[first + row0 + (i + r) * step] = mean[r] + rest[r];
            if (t == 0 && p.rstd) p.rstd[first + row0 + (i + r) * step] = rstd[r];
            if (!p.y) continue;
            const uint64_t scale = both(rstd[r]), off = both(-rest[r] * rstd[r]), m = both(-mean[r]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == U - 1 && !last) continue;
                Eight o = ring.read(i + r, 0, u, t, team);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t d = add_f32x2(o.v[k], m);
                    o.v[k] = fma_f32x2(REST ? fma_f32x2(d, scale, off) : mul_f32x2(d, scale), w[u].v[k], b[u].v[k]);
                }
                put_pairs<T>(y + col<true>(u, 0, t, team), o);
            }
            y += along;
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) fill(i + r + ST);  // the slots just read
    }
    wait_but<0>();
}

// The backward pass with a ring; a row is read from it once for the sums and once for dx.
template <typename T, typename W, int U, int ST, int RB, int MT, int MB, bool SUMS>
__global__ void __launch_bounds__(MT, MB) layer_norm_ring_backward_kernel(const LnParams p) {
    __shared__ float red[2 * RB][MT / 32];
    __shared__ float joint[2 * RB];
    extern __shared__ __align__(16) unsigned char smem[];
    const int t = threadIdx.x, team = blockDim.x, warps = team >> 5, lane = t & 31, warp = t >> 5;
    const int step = gridDim.x * blockDim.y, row0 = blockIdx.x * blockDim.y + threadIdx.y;
    const long long first = (long long)blockIdx.y * p.rows;
    const Ring<T, U, ST, true> ring(smem, team);
    const bool last = col<true>(U - 1, 0, t, team) < p.dim;  // (all groups before it are whole)
    const int mine = row0 < p.rows ? (p.rows - row0 + step - 1) / step : 0;  // rows of this team
    const T* next_x = static_cast<const T*>(p.x) + (first + row0) * p.stride_x;
    const T* next_dy = static_cast<const T*>(p.dy) + (first + row0) * p.stride_dy;
    const long long ahead_x = step * p.stride_x, ahead_dy = step * p.stride_dy, along = (long long)step * p.dim;
    auto fill = [&](int i) {
        if (i < mine) {
            ring.fill(i, 0, next_x, last, t, team);
            ring.fill(i, 1, next_dy, last, t, team);
        }
        next_x += ahead_x;
        next_dy += ahead_dy;
        commit();
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) fill(i);
    T* dx = static_cast<T*>(p.dx) + (first + row0) * p.dim;
    Eight w[U], dw[U], db[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) dw[u].v[k] = db[u].v[k] = 0;
        if (u < U - 1 || last) w[u] = get_pairs<W>(p.w, blockIdx.y * p.stride_w, col<true>(u, 0, t, team), 1.f, p.add);
    }
    const float per_row = 1.f / (float)p.dim;
    float nm[RB], nr[RB];
    auto stats = [&](int i) {
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const long long row = first + row0 + (i + r) * step;
            nm[r] = i + r < mine ? __ldg(p.mean + row) : 0.f;
            nr[r] = i + r < mine ? __ldg(p.rstd + row) : 0.f;
        }
    };
    stats(0);
    for (int i = 0; i < mine; i += RB) {
        wait_but<ST - RB>();
        float mean[RB], rstd[RB], s[2 * RB];
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            s[2 * r] = s[2 * r + 1] = 0.f;
            mean[r] = nm[r], rstd[r] = nr[r];
            if (i + r >= mine) continue;  // (its slot holds an older row)
            const uint64_t scale = both(nr[r]), m = both(-nm[r]);
            uint64_t a0 = 0, a1 = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == U - 1 && !last) continue;
                const Eight xv = ring.read(i + r, 0, u, t, team), dv = ring.read(i + r, 1, u, t, team);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t h = mul_f32x2(add_f32x2(xv.v[k], m), scale), g = dv.v[k];
                    if constexpr (SUMS) {
                        dw[u].v[k] = fma_f32x2(g, h, dw[u].v[k]);
                        db[u].v[k] = add_f32x2(g, db[u].v[k]);
                    }
                    const uint64_t gw = mul_f32x2(g, w[u].v[k]);
                    a0 = add_f32x2(gw, a0);
                    a1 = fma_f32x2(gw, h, a1);
                }
            }
            s[2 * r] = sum_pairs(a0);
            s[2 * r + 1] = sum_pairs(a1);
        }
        stats(i + RB);
        const float ws = warp_sums<2 * RB>(s);
        float m[2 * RB];
        if (warps == 1) {
#pragma unroll
            for (int r = 0; r < 2 * RB; ++r) m[r] = __shfl_sync(0xffffffffu, ws, r * (16 / RB)) * per_row;
        } else {
            if ((lane & (16 / RB - 1)) == 0) red[lane / (16 / RB)][warp] = ws;
            __syncthreads();
            for (int r = warp; r < 2 * RB; r += warps) {
                const float one[1] = {lane < warps ? red[r][lane] : 0.f};
                const float all = warp_sums<1>(one);
                if (lane == 0) joint[r] = all * per_row;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2 * RB; ++r) m[r] = joint[r];
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            if (i + r >= mine || !p.dx) continue;
            // v - mean(v) - xh mean(v xh) as a line in x - mean beside v
            const uint64_t scale = both(rstd[r]), c1 = both(-rstd[r] * m[2 * r + 1]), c0 = both(-m[2 * r]), off = both(-mean[r]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == U - 1 && !last) continue;
                const Eight xv = ring.read(i + r, 0, u, t, team);
                Eight o = ring.read(i + r, 1, u, t, team);
#pragma unroll
                for (int k = 0; k < 4; ++k) o.v[k] = mul_f32x2(fma_f32x2(o.v[k], w[u].v[k], fma_f32x2(add_f32x2(xv.v[k], off), c1, c0)), scale);
                put_pairs<T>(dx + col<true>(u, 0, t, team), o);
            }
            dx += along;
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) fill(i + r + ST);  // the slots just read
    }
    wait_but<0>();
    if constexpr (SUMS) {
        __syncthreads();  // the ring's memory takes the teams' sums
        float fw[U][8], fb[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 a = unpack_f32x2(dw[u].v[k]), c = unpack_f32x2(db[u].v[k]);
                fw[u][2 * k] = a.x; fw[u][2 * k + 1] = a.y;
                fb[u][2 * k] = c.x; fb[u][2 * k + 1] = c.y;
            }
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) on[u] = u < U - 1 || last;
        leave_sums<U, true>(p, fw, fb, on, reinterpret_cast<float*>(smem));
    }
}

// Sums of the CTAs' partial rows: a CTA takes 32 columns, its warps every kSumLanes-th partial row.
constexpr int kSumLanes = 16;
template <typename W>
__global__ void __launch_bounds__(32 * kSumLanes) layer_norm_sums_kernel(const float* part, int parts, int dim, W* dw, W* db) {
    __shared__ float sum[kSumLanes][32];
    const int c = blockIdx.x * 32 + threadIdx.x;  // of 2 dim: first the weight's, then the bias'
    const float* p = part + (long long)blockIdx.y * parts * 2 * dim;
    float s = 0.f;
    if (c < 2 * dim) {
#pragma unroll 8
        for (int i = threadIdx.y; i < parts; i += kSumLanes) s += __ldg(p + (long long)i * 2 * dim + c);
    }
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < 2 * dim) {
#pragma unroll
        for (int i = 1; i < kSumLanes; ++i) s += sum[i][threadIdx.x];
        W* out = c < dim ? dw : db;
        if (out) st1<W>(out + (long long)blockIdx.y * dim + (c < dim ? c : c - dim), s);
    }
}

// How a call is laid out: threads of a team, teams of a CTA, groups of eight columns per thread, slots of a team's ring (0:
// no ring), dynamic shared memory, CTAs per group of rows.
struct Shape {
    int team, teams, u, st, smem, ctas;
};
constexpr int kSmemPerSm = 220 * 1024;
int ctas_per_group(int resident, int groups) {
    const int sms = nb_num_sms(), per = resident * (sms > 0 ? sms : 148) / groups;
    return per < 1 ? 1 : per;
}
// `ring`: the rows are whole 16-byte pieces.  The ring has 8 slots while two CTAs of it (three in the backward pass) fit an
// SM, else 4; rows too long for that (over 27 KB a slot: 13 K channels of 16 bits in the backward pass) go to the kernel without one.
Shape shape_of(int groups, int rows, int dim, int size, bool backward, bool ring) {
    Shape s;
    const int eights = (dim + 7) / 8;
    if (dim <= 512) {  // a warp per row: no barriers
        s.u = eights <= 32 ? 1 : 2;
        s.team = 32;
        s.teams = 8;
    } else {
        s.u = eights <= 256 ? 1 : eights <= 1024 ? 2 : 4;
        s.team = ((eights + s.u - 1) / s.u + 31) / 32 * 32;
        s.teams = 1;
    }
    const int slot = s.team * s.teams * s.u * 8 * size * (backward ? 2 : 1);
    s.st = !ring ? 0 : slot * 8 <= kSmemPerSm / (backward ? 3 : 2) ? 8 : slot * 4 <= kSmemPerSm ? 4 : 0;
    s.smem = s.st * slot;
    const int joined = backward && s.teams > 1 ? s.teams * 2 * dim * 4 : 0;  // at most 8 x 2 x 512 x 4 = 32 KB
    if (s.smem < joined) s.smem = joined;
    // CTAs per group of rows, at most: what an SM can hold by threads and shared memory (run() takes what it does hold)
    const int threads = s.team * s.teams;
    int resident = (backward ? 768 : 1024) / threads;
    if (s.smem && resident > kSmemPerSm / (s.smem + 2048)) resident = kSmemPerSm / (s.smem + 2048);
    if (resident < 1) resident = 1;
    const int want = (rows + s.teams - 1) / s.teams, per = ctas_per_group(resident, groups);
    s.ctas = want < per ? want : per;
    return s;
}

template <typename K>
int run(K kernel, const LnParams& p, Shape& s, int groups, cudaStream_t st) {
    if (s.smem > 40 * 1024)  // 48 KB without asking, the static arrays among them
        NB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, s.smem));
    // one wave: a second one would leave most SMs idle while it runs
    int resident = 0;
    NB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, s.team * s.teams, s.smem));
    const int per = ctas_per_group(resident, groups);
    if (s.ctas > per) s.ctas = per;
    kernel<<<dim3(s.ctas, groups), dim3(s.team, s.teams), s.smem, st>>>(p);
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
// MT, MB: threads of a CTA at most and CTAs per SM at least, which give the kernels' registers
template <typename T, typename W, int U, int MT, int MB>
int launch(const LnParams& p, Shape& s, int groups, bool backward, cudaStream_t st) {
    if (!backward) {
        if (s.st == 8) return run(layer_norm_ring_kernel<T, W, U, 8, 4, MT, MB>, p, s, groups, st);
        if (s.st == 4) return run(layer_norm_ring_kernel<T, W, U, 4, 2, MT, MB>, p, s, groups, st);
        return run(layer_norm_kernel<T, W, U>, p, s, groups, st);
    }
    if (p.part) {
        if (s.st == 8) return run(layer_norm_ring_backward_kernel<T, W, U, 8, 2, MT, MB, true>, p, s, groups, st);
        if (s.st == 4) return run(layer_norm_ring_backward_kernel<T, W, U, 4, 2, MT, MB, true>, p, s, groups, st);
        return run(layer_norm_backward_kernel<T, W, U, true>, p, s, groups, st);
    }
    if (s.st == 8) return run(layer_norm_ring_backward_kernel<T, W, U, 8, 2, MT, MB, false>, p, s, groups, st);
    if (s.st == 4) return run(layer_norm_ring_backward_kernel<T, W, U, 4, 2, MT, MB, false>, p, s, groups, st);
    return run(layer_norm_backward_kernel<T, W, U, false>, p, s, groups, st);
}
template <typename T, typename W>
int launch(const LnParams& p, Shape& s, int groups, bool backward, cudaStream_t st) {
    switch (s.u) {
        case 1: return launch<T, W, 1, 256, 3>(p, s, groups, backward, st);
        case 2: return s.team <= 320 ? launch<T, W, 2, 320, 2>(p, s, groups, backward, st) : launch<T, W, 2, 512, 1>(p, s, groups, backward, st);
        default: return launch<T, W, 4, 512, 1>(p, s, groups, backward, st);
    }
}
int launch(const LnParams& p, Shape& s, const nb_layer_norm_args* a, bool backward, cudaStream_t st) {
    if (a->dtype == NB_DTYPE_FP32) return launch<float, float>(p, s, a->groups, backward, st);
    if (a->dtype == NB_DTYPE_BF16)
        return a->w_fp32 ? launch<__nv_bfloat16, float>(p, s, a->groups, backward, st)
                         : launch<__nv_bfloat16, __nv_bfloat16>(p, s, a->groups, backward, st);
    return a->w_fp32 ? launch<__half, float>(p, s, a->groups, backward, st) : launch<__half, __half>(p, s, a->groups, backward, st);
}
int size_of(const nb_layer_norm_args* a) { return a->dtype == NB_DTYPE_FP32 ? 4 : 2; }

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
    if (groups <= 0 || rows <= 0 || dim <= 0 || dim > NB_LAYER_NORM_MAX_DIM) return 0;
    const int size = dtype == NB_DTYPE_FP32 ? 4 : 2;  // with or without a ring: alignment is not known here
    const int a = nb::shape_of(groups, rows, dim, size, true, false).ctas, b = nb::shape_of(groups, rows, dim, size, true, true).ctas;
    return (int64_t)(a > b ? a : b) * groups * 2 * dim * 4;
}

extern "C" int nb_layer_norm(const nb_layer_norm_args* a, void* stream) {
    using namespace nb;
    if (int rc = check(a)) return rc;
    if (a->rows == 0) return NB_OK;
    NB_REQUIRE(a->x);
    const int per = 16 / size_of(a);
    const bool ring = a->dim % 8 == 0 && aligned16(a->x) && aligned16(a->y) && a->stride_x % per == 0 && vec_w(a, a->w) && vec_w(a, a->b);
    Shape s = shape_of(a->groups, a->rows, a->dim, size_of(a), false, ring);
    return launch(params_of(a), s, a, false, static_cast<cudaStream_t>(stream));
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
    const int per = 16 / size_of(a);
    const bool ring = a->dim % 8 == 0 && aligned16(a->x) && aligned16(a->dy) && aligned16(a->dx) && a->stride_x % per == 0 &&
                      a->stride_dy % per == 0 && vec_w(a, a->w);
    Shape s = shape_of(a->groups, a->rows, a->dim, size_of(a), true, ring);
    LnParams p = params_of(a);
    if (sums) {
        NB_REQUIRE(a->workspace && aligned16(a->workspace));
        if (a->workspace_bytes < (int64_t)s.ctas * a->groups * 2 * a->dim * 4)
            return fail_with(NB_ERR_INVALID, "workspace smaller than nb_layer_norm_workspace_bytes()");
        p.part = static_cast<float*>(a->workspace);
    }
    if (int rc = launch(p, s, a, true, st)) return rc;
    if (!sums) return NB_OK;
    const dim3 grid((2 * a->dim + 31) / 32, a->groups), block(32, kSumLanes);
    if (a->w_fp32 || a->dtype == NB_DTYPE_FP32)
        layer_norm_sums_kernel<float><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<float*>(a->dw), static_cast<float*>(a->db));
    else if (a->dtype == NB_DTYPE_BF16)
        layer_norm_sums_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<__nv_bfloat16*>(a->dw), static_cast<__nv_bfloat16*>(a->db));
    else
        layer_norm_sums_kernel<__half><<<grid, block, 0, st>>>(p.part, s.ctas, a->dim, static_cast<__half*>(a->dw), static_cast<__half*>(a->db));
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
