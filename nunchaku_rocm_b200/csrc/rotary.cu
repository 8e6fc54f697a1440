// Rotary positions with several axes (time, height, width), straight from position ids.
//
// The rotary channels of a head are split over the axes: axis a owns d_a of them, d_a / 2 channel pairs.  Pair j of an axis
// turns by pos_a * theta^(-2 j / d_a) radians:
//
//     (u, v) -> (u cos t - v sin t, u sin t + v cos t)
//
// and its backward pass is the rotation by -t.  A pair is two neighbouring channels (interleaved) or the channels j and
// j + R/2 of the R rotary ones (half-split); channels behind the R rotary ones pass through.
//
// The angle is taken in TURNS in fp64 (position times rate), reduced to an eighth of a turn there and only then rounded to
// fp32: the rounding is 2^-28 of a turn whatever the position, where an fp32 angle of a far position has lost its fraction.
// One (cos, sin) per token and pair goes through shared memory to all heads of Q and K, so the fp64 work is 1 / (heads of Q
// and K) of the pairs.
//
// Bound: HBM.  Q and K are read once and written once (16-byte accesses when the layout allows), the ids are 4 to 12 bytes
// per token.  Measured on a B200: Q and K of 4608 tokens and 24 + 24 heads of 128 as views of a packed QKV, bf16, 25.2 us (4.5
// TB/s; a copy of as many bytes takes 24.3); 32986 tokens, 24 + 8 heads, halves paired, fp16, 85 us (6.4 TB/s).
#include <math.h>

#include "nb_common.cuh"

namespace nb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTok = 16;  // tokens per CTA

// n / d for 0 <= n < 2^31 by a multiplication and a shift (Granlund and Montgomery, Division by Invariant Integers using
// Multiplication, 1994)
struct FastDiv {
    uint32_t d, mul, shift;
};
FastDiv make_fastdiv(uint32_t d) {
    FastDiv f = {d, 0, 0};
    while ((1ull << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}
__device__ __forceinline__ uint32_t fastdiv(uint32_t n, const FastDiv& f) {
    const uint32_t hi = __umulhi(n, f.mul);
    return (uint32_t)(((uint64_t)hi + n) >> f.shift);
}

struct RotParams {
    const void* q; const void* k; void* qo; void* ko;
    const void* ids;
    long long sq_b, sq_s, sq_h, sk_b, sk_s, sk_h;  // elements; the outputs are contiguous (B, S, heads, D)
    long long si_b, si_s, si_a;
    int S, H, Hk, D, pairs, ids_type;
    uint32_t rows;        // B * S
    int tok;              // tokens per CTA
    int units;            // work items per head
    int rot_units;        // the first of them rotate, the rest copy
    float sign;           // +1, or -1 for the inverse rotation
    FastDiv div_units, div_heads, div_s;
    nb_rotary_ladder ladder;
};

__device__ __forceinline__ double load_id(const void* ids, int type, long long i) {
    switch (type) {
        case NB_IDS_F32: return (double)__ldg(static_cast<const float*>(ids) + i);
        case NB_IDS_I32: return (double)__ldg(static_cast<const int*>(ids) + i);
        case NB_IDS_I64: return (double)__ldg(static_cast<const long long*>(ids) + i);
        default: return __ldg(static_cast<const double*>(ids) + i);
    }
}

__device__ __forceinline__ int axis_of(const nb_rotary_ladder& l, int pair) {
    int a = 0;
#pragma unroll
    for (int i = 0; i < NB_ROTARY_MAX_AXES - 1; ++i) a += (i + 1 < l.n_axes && pair >= l.pair_end[i]) ? 1 : 0;
    return a;
}

// (cos, sin) of `turns` whole turns, rounded once.  Whole turns and then the nearest quarter are taken off; what is left, an
// angle y of at most pi / 4, goes through the Taylor series (first terms left out: y^13 / 13! and y^12 / 12!, under 2^-33), and
// the quarter turns it by swaps and signs.  All in fp64, whose rate here is half of fp32's: in fp32 the table was 2.5e-8 off on
// the average, where one rounding of the true values is 1.9e-8, for the same time.  (The library's sincospi reduces once more
// and took twice as long; where there are few heads per token the angles are what the kernel waits for.)
__device__ __forceinline__ float2 cos_sin_turns(double turns) {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double part = turns - __dadd_rn(__dadd_rn(turns, kRound), -kRound);  // [-1/2, 1/2]
    const float quarter = rintf(4.f * (float)part);
    const double y = fma(-0.25, (double)quarter, part) * 6.283185307179586476925, z = y * y;
    const double s3 = fma(z, fma(z, fma(z, fma(z, -1. / 39916800., 1. / 362880.), -1. / 5040.), 1. / 120.), -1. / 6.);
    const double c2 = fma(z, fma(z, fma(z, fma(z, -1. / 3628800., 1. / 40320.), -1. / 720.), 1. / 24.), -0.5);
    const float s = (float)fma(y * z, s3, y), c = (float)fma(z, c2, 1.);
    const int n = (int)quarter & 3;
    const float cs = (n & 1) ? s : c, sn = (n & 1) ? c : s;
    return make_float2((n == 1 || n == 2) ? -cs : cs, (n >= 2) ? -sn : sn);
}

template <typename T>
struct Vec;  // 16 bytes of T as fp32
template <>
struct Vec<float> {
    static constexpr int N = 4;
    __device__ static void widen(const uint4& r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    }
    __device__ static uint4 narrow(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <typename T>
struct Vec16 {
    static constexpr int N = 8;
    __device__ static void widen(const uint4& r, float (&v)[8]) {
        float2 f;
        f = unpack2<T>(r.x); v[0] = f.x; v[1] = f.y;
        f = unpack2<T>(r.y); v[2] = f.x; v[3] = f.y;
        f = unpack2<T>(r.z); v[4] = f.x; v[5] = f.y;
        f = unpack2<T>(r.w); v[6] = f.x; v[7] = f.y;
    }
    __device__ static uint4 narrow(const float (&v)[8]) {
        return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
};
template <> struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16> {};
template <> struct Vec<__half> : Vec16<__half> {};

template <typename T> __device__ __forceinline__ float load1(const T* p) { return to_f32<T>(*p); }
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ void store1(T* p, float v) { *p = from_f32<T>(v); }
template <> __device__ __forceinline__ void store1<float>(float* p, float v) { *p = v; }

// where item `i` of a CTA's tokens lies
struct Item {
    const void* src;
    void* dst;
    int tok, unit;
};
template <typename T>
__device__ __forceinline__ Item locate(const RotParams& p, uint32_t row0, uint32_t i) {
    const uint32_t th = fastdiv(i, p.div_units);  // token * heads + head
    Item it;
    it.unit = (int)(i - th * p.div_units.d);
    it.tok = (int)fastdiv(th, p.div_heads);
    const int head = (int)(th - (uint32_t)it.tok * p.div_heads.d);
    const uint32_t row = row0 + it.tok;
    const uint32_t b = fastdiv(row, p.div_s), s = row - b * p.div_s.d;
    if (head < p.H) {
        it.src = static_cast<const T*>(p.q) + (b * p.sq_b + s * p.sq_s + head * p.sq_h);
        it.dst = static_cast<T*>(p.qo) + ((long long)row * p.H + head) * p.D;
    } else {
        it.src = static_cast<const T*>(p.k) + (b * p.sk_b + s * p.sk_s + (head - p.H) * p.sk_h);
        it.dst = static_cast<T*>(p.ko) + ((long long)row * p.Hk + (head - p.H)) * p.D;
    }
    return it;
}

// W neighbouring channels (4 or 8 bytes) in one access
template <typename T, int W>
struct alignas(sizeof(T) * W) Pack {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ Pack<T, W> load_pack(const T* at) {
    static_assert(sizeof(T) * W == 4 || sizeof(T) * W == 8, "others go by 16 bytes or one by one");
    Pack<T, W> p;
    if constexpr (sizeof(T) * W == 8) *reinterpret_cast<uint2*>(&p) = __ldg(reinterpret_cast<const uint2*>(at));
    else *reinterpret_cast<uint32_t*>(&p) = __ldg(reinterpret_cast<const uint32_t*>(at));
    return p;
}

// W channels per access.  16 bytes (VEC): an item is 16 bytes of a head (interleaved), two 16-byte pieces R/2 apart (HALF), or
// 16 bytes that pass through; with SHARED, the last rotated pairs and the first channels that pass through are in one piece.
// HALF with fewer: two pieces of W channels, or W that pass through.  One: a channel pair, or one channel that passes through,
// for every size and alignment.  Measured, 9000 tokens of 24 + 24 heads, bf16: halves of 36 of 72 channels 67 us with single
// channels, 36 with four; 63 interleaved pairs of 128 channels 116 us pair by pair, 51 with a shared piece (64 pairs, without the
// tests that a shared piece needs: 43).
template <typename T, bool HALF, int W, bool SHARED>
__global__ void __launch_bounds__(kThreads, HALF ? 4 : 5) rotary_kernel(const __grid_constant__ RotParams p) {
    extern __shared__ float2 cs[];  // [tok][cols]
    constexpr bool VEC = W * sizeof(T) == 16;
    const uint32_t row0 = blockIdx.x * (uint32_t)p.tok;
    const int ntok = (int)min((uint32_t)p.tok, p.rows - row0);
    const uint32_t items = (uint32_t)ntok * (p.H + p.Hk) * p.units;

    // The first items' loads are issued before the angles are computed, so that they travel meanwhile.
    constexpr int N = Vec<T>::N;
    constexpr int PER = HALF ? W : VEC ? N / 2 : 1;  // pairs of an item
    constexpr int AHEAD = HALF ? 4 : 3;
    const int steps = (p.pairs + PER - 1) / PER, cols = steps * PER;  // (a shared piece's places behind the last pair are not read)
    Item it[AHEAD];
    uint4 r0[AHEAD], r1[AHEAD];
    auto fetch = [&](uint32_t first) {
        if constexpr (VEC) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const uint32_t i = first + a * kThreads;
                if (i >= items) continue;
                it[a] = locate<T>(p, row0, i);
                const T* src = static_cast<const T*>(it[a].src);
                if (HALF && it[a].unit < p.rot_units) {
                    r0[a] = __ldg(reinterpret_cast<const uint4*>(src + it[a].unit * N));
                    r1[a] = __ldg(reinterpret_cast<const uint4*>(src + p.pairs + it[a].unit * N));
                } else {
                    const int at = HALF ? 2 * p.pairs + (it[a].unit - p.rot_units) * N : it[a].unit * N;
                    r0[a] = __ldg(reinterpret_cast<const uint4*>(src + at));
                }
            }
        }
    };
    fetch(threadIdx.x);

    // a thread keeps its pair (one rate, one axis) and walks over the tokens
    const int pair = threadIdx.x % p.pairs, per = kThreads / p.pairs;
    if (threadIdx.x < per * p.pairs) {
        const double rate = p.ladder.turns[pair];
        const long long axis = axis_of(p.ladder, pair) * p.si_a;
        // the PER pairs of an item lie `steps` apart, so that the lanes of a warp read neighbouring words
        const int at = (pair % PER) * steps + pair / PER;
        for (int tok = threadIdx.x / p.pairs; tok < ntok; tok += per) {
            const uint32_t row = row0 + tok, b = fastdiv(row, p.div_s), s = row - b * p.div_s.d;
            float2 v = cos_sin_turns(load_id(p.ids, p.ids_type, b * p.si_b + s * p.si_s + axis) * rate);
            v.y *= p.sign;
            cs[tok * cols + at] = v;
        }
    }
    __syncthreads();

    if constexpr (VEC) {
        for (uint32_t first = threadIdx.x; first < items; first += AHEAD * kThreads) {
            if (first != threadIdx.x) fetch(first);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (first + a * kThreads >= items) continue;
                T* dst = static_cast<T*>(it[a].dst);
                const float2* w = cs + it[a].tok * cols;
                if (it[a].unit >= p.rot_units) {
                    const int at = HALF ? 2 * p.pairs + (it[a].unit - p.rot_units) * N : it[a].unit * N;
                    *reinterpret_cast<uint4*>(dst + at) = r0[a];
                } else if constexpr (HALF) {
                    float u[N], v[N], x[N], y[N];
                    Vec<T>::widen(r0[a], u);
                    Vec<T>::widen(r1[a], v);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float2 c = w[j * steps + it[a].unit];
                        x[j] = u[j] * c.x - v[j] * c.y;
                        y[j] = u[j] * c.y + v[j] * c.x;
                    }
                    *reinterpret_cast<uint4*>(dst + it[a].unit * N) = Vec<T>::narrow(x);
                    *reinterpret_cast<uint4*>(dst + p.pairs + it[a].unit * N) = Vec<T>::narrow(y);
                } else {
                    float u[N], x[N];
                    Vec<T>::widen(r0[a], u);
                    const int left = p.pairs - it[a].unit * PER;  // pairs of this piece that turn
#pragma unroll
                    for (int j = 0; j < N / 2; ++j) {
                        if (SHARED && j >= left) {
                            x[2 * j] = u[2 * j];
                            x[2 * j + 1] = u[2 * j + 1];
                            continue;
                        }
                        const float2 c = w[j * steps + it[a].unit];
                        x[2 * j] = u[2 * j] * c.x - u[2 * j + 1] * c.y;
                        x[2 * j + 1] = u[2 * j] * c.y + u[2 * j + 1] * c.x;
                    }
                    *reinterpret_cast<uint4*>(dst + it[a].unit * N) = Vec<T>::narrow(x);
                }
            }
        }
    } else if constexpr (W > 1) {
        static_assert(HALF, "interleaved pairs go by 16 bytes or one by one");
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
            const Item m = locate<T>(p, row0, i);
            const T* src = static_cast<const T*>(m.src);
            T* dst = static_cast<T*>(m.dst);
            if (m.unit >= p.rot_units) {
                const int at = 2 * p.pairs + (m.unit - p.rot_units) * W;
                *reinterpret_cast<Pack<T, W>*>(dst + at) = load_pack<T, W>(src + at);
                continue;
            }
            const int at = m.unit * W;
            const float2* w = cs + m.tok * cols + m.unit;
            const Pack<T, W> u = load_pack<T, W>(src + at), v = load_pack<T, W>(src + p.pairs + at);
            Pack<T, W> x, y;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float2 c = w[j * steps];
                const float a = load1<T>(u.v + j), b = load1<T>(v.v + j);
                store1<T>(x.v + j, a * c.x - b * c.y);
                store1<T>(y.v + j, a * c.y + b * c.x);
            }
            *reinterpret_cast<Pack<T, W>*>(dst + at) = x;
            *reinterpret_cast<Pack<T, W>*>(dst + p.pairs + at) = y;
        }
    } else {
        for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
            const Item m = locate<T>(p, row0, i);
            const T* src = static_cast<const T*>(m.src);
            T* dst = static_cast<T*>(m.dst);
            if (m.unit >= p.rot_units) {
                const int at = 2 * p.pairs + (m.unit - p.rot_units);
                dst[at] = src[at];
            } else {
                const int at = HALF ? m.unit : 2 * m.unit, to = HALF ? m.unit + p.pairs : at + 1;
                const float2 c = cs[m.tok * cols + m.unit];
                const float u = load1<T>(src + at), v = load1<T>(src + to);
                store1<T>(dst + at, u * c.x - v * c.y);
                store1<T>(dst + to, u * c.y + v * c.x);
            }
        }
    }
}

// (rows, pairs) of (sin, cos) in fp32: a thread keeps one pair (one rate) and walks over the rows
__global__ void __launch_bounds__(kThreads) rotary_table_kernel(const __grid_constant__ RotParams p, float2* out) {
    const int pair = threadIdx.x % p.pairs, lane = threadIdx.x / p.pairs;
    const int per = kThreads / p.pairs;  // rows a CTA works on at a time
    if (lane >= per) return;
    const double rate = p.ladder.turns[pair];
    const int axis = axis_of(p.ladder, pair);
    for (uint32_t row = blockIdx.x * per + lane; row < p.rows; row += gridDim.x * per) {
        const uint32_t b = fastdiv(row, p.div_s), s = row - b * p.div_s.d;
        const float2 v = cos_sin_turns(load_id(p.ids, p.ids_type, b * p.si_b + s * p.si_s + axis * p.si_a) * rate);
        out[(long long)row * p.pairs + pair] = make_float2(v.y, v.x);
    }
}

template <typename T, bool HALF, int W, bool SHARED = false>
int launch_w(const RotParams& p, cudaStream_t s) {
    const uint32_t blocks = (p.rows + p.tok - 1) / p.tok;
    const size_t smem = sizeof(float2) * (size_t)p.tok * ((p.pairs + 7) / 8 * 8);  // at most 16 tokens x 128 pairs x 8 bytes = 16 KB
    rotary_kernel<T, HALF, W, SHARED><<<blocks, kThreads, smem, s>>>(p);
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
template <typename T>
int launch_rot(const RotParams& p, bool half, int w, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (half) {
        if (w == N) return launch_w<T, true, N>(p, s);
        if (w == N / 2) return launch_w<T, true, N / 2>(p, s);
        if constexpr (N > 4) if (w == 2) return launch_w<T, true, 2>(p, s);
        return launch_w<T, true, 1>(p, s);
    }
    if (w < N) return launch_w<T, false, 1>(p, s);
    return 2 * p.pairs % N ? launch_w<T, false, N, true>(p, s) : launch_w<T, false, N>(p, s);
}

bool good_ladder(const nb_rotary_ladder* l) {
    if (!l || l->n_axes < 1 || l->n_axes > NB_ROTARY_MAX_AXES) return false;
    int last = 0;
    for (int i = 0; i < l->n_axes; ++i) {
        if (l->pair_end[i] <= last || l->pair_end[i] > NB_ROTARY_MAX_PAIRS) return false;
        last = l->pair_end[i];
    }
    return true;
}

}  // namespace
}  // namespace nb

extern "C" int nb_rotary_ladder_init(nb_rotary_ladder* l, const int32_t* axes_dim, int32_t n_axes, double theta) {
    using namespace nb;
    NB_REQUIRE(l && axes_dim && n_axes >= 1 && n_axes <= NB_ROTARY_MAX_AXES && theta > 0 && isfinite(theta));
    int at = 0;
    for (int i = 0; i < n_axes; ++i) {
        const int d = axes_dim[i];
        NB_REQUIRE(d > 0 && d % 2 == 0 && d <= 2 * (NB_ROTARY_MAX_PAIRS - at));
        for (int j = 0; j < d / 2; ++j) l->turns[at++] = pow(theta, -2.0 * j / d) / 6.283185307179586476925;
        l->pair_end[i] = at;
    }
    l->n_axes = n_axes;
    return NB_OK;
}

extern "C" int nb_rotary_axes(const nb_rotary_args* a, const nb_rotary_ladder* l, void* stream) {
    using namespace nb;
    NB_REQUIRE(a && good_ladder(l));
    NB_REQUIRE(a->B >= 0 && a->S >= 0 && a->H > 0 && a->Hk >= 0 && a->D > 0);
    NB_REQUIRE(a->ids_type >= NB_IDS_F32 && a->ids_type <= NB_IDS_F64);
    NB_REQUIRE(a->dtype == NB_DTYPE_BF16 || a->dtype == NB_DTYPE_FP16 || a->dtype == NB_DTYPE_FP32);
    const int pairs = l->pair_end[l->n_axes - 1];
    if (2 * pairs > a->D) return fail_with(NB_ERR_INVALID, "the axes have more channels than a head");
    const long long rows = (long long)a->B * a->S;
    if (rows == 0) return NB_OK;
    NB_REQUIRE(a->q && a->q_out && a->ids && (a->Hk == 0 || (a->k && a->k_out)));
    const long long heads = (long long)a->H + a->Hk;
    if (rows > 0x7fffffffll || heads * a->D > (1 << 26)) return fail_with(NB_ERR_TOO_LARGE, "more than 2^31 rows or 2^26 channels per row");
    const int size = a->dtype == NB_DTYPE_FP32 ? 4 : 2, n = 16 / size;
    RotParams p = {};
    p.q = a->q; p.k = a->k; p.qo = a->q_out; p.ko = a->k_out; p.ids = a->ids;
    p.sq_b = a->stride_qb; p.sq_s = a->stride_qs; p.sq_h = a->stride_qh;
    p.sk_b = a->stride_kb; p.sk_s = a->stride_ks; p.sk_h = a->stride_kh;
    p.si_b = a->stride_ib; p.si_s = a->stride_is; p.si_a = a->stride_ia;
    p.S = a->S; p.H = a->H; p.Hk = a->Hk; p.D = a->D; p.pairs = pairs; p.ids_type = a->ids_type;
    p.rows = (uint32_t)rows;
    p.sign = a->inverse ? -1.f : 1.f;
    p.ladder = *l;
    // channels per access: the rows of all tensors start on its multiples, and it divides a head and, where the pairs are split,
    // each half
    const auto fits = [&](int w) {
        const auto on = [&](const void* at, int64_t b, int64_t s, int64_t h) {
            return reinterpret_cast<uintptr_t>(at) % (w * size) == 0 && b % w == 0 && s % w == 0 && h % w == 0;
        };
        return a->D % w == 0 && (!a->half || pairs % w == 0) && on(a->q, a->stride_qb, a->stride_qs, a->stride_qh) && on(a->q_out, 0, 0, 0) &&
               (a->Hk == 0 || (on(a->k, a->stride_kb, a->stride_ks, a->stride_kh) && on(a->k_out, 0, 0, 0)));
    };
    int w = n;
    while (w > 1 && !fits(w)) w /= 2;
    if (!a->half && w < n) w = 1;
    if (a->half || w < n) {
        p.rot_units = a->half ? pairs / w : pairs;
        p.units = p.rot_units + (a->D - 2 * pairs) / w;
    } else {
        p.rot_units = (2 * pairs + n - 1) / n;
        p.units = a->D / n;
    }
    // Tokens per CTA: about four items per thread, but never so many that the CTAs do not cover the SMs.
    int sms = nb_num_sms();
    if (sms <= 0) sms = 148;
    long long tok = (4ll * kThreads) / (heads * p.units);
    const long long spread = rows / (2ll * sms);
    if (tok > spread) tok = spread;
    p.tok = (int)(tok < 1 ? 1 : tok > kMaxTok ? kMaxTok : tok);
    p.div_units = make_fastdiv(p.units);
    p.div_heads = make_fastdiv((uint32_t)heads);
    p.div_s = make_fastdiv(a->S);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == NB_DTYPE_BF16) return launch_rot<__nv_bfloat16>(p, a->half, w, s);
    if (a->dtype == NB_DTYPE_FP16) return launch_rot<__half>(p, a->half, w, s);
    return launch_rot<float>(p, a->half, w, s);
}

extern "C" int nb_rotary_table(const void* ids, int32_t ids_type, int32_t B, int32_t S, int64_t stride_ib, int64_t stride_is,
                               int64_t stride_ia, float* out, const nb_rotary_ladder* l, void* stream) {
    using namespace nb;
    NB_REQUIRE(good_ladder(l) && B >= 0 && S >= 0 && ids_type >= NB_IDS_F32 && ids_type <= NB_IDS_F64);
    const long long rows = (long long)B * S;
    if (rows == 0) return NB_OK;
    NB_REQUIRE(ids && out && (reinterpret_cast<uintptr_t>(out) & 7) == 0);
    if (rows > 0x7fffffffll) return fail_with(NB_ERR_TOO_LARGE, "more than 2^31 rows");
    RotParams p = {};
    p.ids = ids; p.ids_type = ids_type;
    p.si_b = stride_ib; p.si_s = stride_is; p.si_a = stride_ia;
    p.S = S; p.rows = (uint32_t)rows;
    p.pairs = l->pair_end[l->n_axes - 1];
    p.div_s = make_fastdiv(S);
    p.ladder = *l;
    const int per = kThreads / p.pairs;  // pairs <= NB_ROTARY_MAX_PAIRS = 128
    const long long want = (rows + per - 1) / per;
    int sms = nb_num_sms();
    if (sms <= 0) sms = 148;
    const int blocks = (int)(want < 8ll * sms ? want : 8ll * sms);
    rotary_table_kernel<<<blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, reinterpret_cast<float2*>(out));
    NB_CUDA_CHECK(cudaGetLastError());
    return NB_OK;
}
