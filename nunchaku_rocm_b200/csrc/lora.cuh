// What the kernels of the batched adapters share: their parameters and how the work is cut into items.
#pragma once

#include <type_traits>

#include "nb_common.cuh"

namespace nb {
namespace lora {

// h and g (fp32 sums, T x R) as the second products' operands: PARTS planes of 16-bit values that add up to them.
// bf16: three parts of eight bits each are the 24 bits of an fp32 value, exactly (two would lose its last eight).
// fp16: two parts of eleven bits and the second one's sign, so 2^-22 of a value is lost at most.  fp16 has neither the values'
// range (scale x x down reaches far beyond 65504) nor, below 2^-14, its own eleven bits (gradients of adapters that have just
// begun to train are that small), so with SCALED a row is divided by a power of two that brings its largest finite value to
// 2^14 .. 2^15, and the T powers stand behind the planes as floats.  A second product over the ranks multiplies its sums by
// them; one over the rows first brings its item's rows to their largest power.  The 22 bits are there down to 2^-17 of a row's
// (an item's) largest value; what is smaller is off by 2^-39 of the largest.
template <typename T>
struct Split {
    static constexpr bool SCALED = std::is_same<T, __half>::value;
    static constexpr int PARTS = SCALED ? 2 : 3;
};
__host__ __device__ inline int parts_of(int dtype) { return dtype == NB_DTYPE_FP16 ? 2 : 3; }
inline bool scaled(int dtype) { return dtype == NB_DTYPE_FP16; }
__host__ __device__ inline long long plane_bytes(int T, int R) { return (long long)T * R * 2; }

// The power of two that divides a row whose largest finite magnitude is `big`; rows of zeros have the smallest.
__device__ __forceinline__ int row_exponent(float big) { return min(max((int)(__float_as_uint(big) >> 23) - 127 - 14, -126), 126); }
__device__ __forceinline__ float exp2_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127
// `f` / 2^e, f a row's power of two and 2^e its item's largest, as a product of two that fp16 holds (down to 2^-44: smaller
// ones leave nothing of a finite value, and an infinite one infinite)
__device__ __forceinline__ void row_ratio(float f, int e, float& a, float& b) {
    const int d = (int)(__float_as_uint(f) >> 23) - 127 - e;
    a = exp2_of(min(max(d, -20), 0));
    b = exp2_of(min(max(d + 20, -24), 0));
}
__device__ __forceinline__ float finite_abs(float v) { return isfinite(v) ? fabsf(v) : 0.f; }

// A pair of values as PARTS words.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[Split<T>::PARTS]) {
#pragma unroll
    for (int i = 0; i < Split<T>::PARTS; ++i) {
        // bf16 takes the upper halves as they are: rounded, the largest fp32 values would be infinite
        part[i] = Split<T>::SCALED ? pack2<T>(x, y) : __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
        const float2 back = unpack2<T>(part[i]);
        // (a value that is not finite is so in the first part alone)
        x = isfinite(back.x) ? x - back.x : 0.f;
        y = isfinite(back.y) ? y - back.y : 0.f;
    }
}

struct LoraParams {
    const void* x;        // shrink: (T, K) operand; expand: base (T, C) or null
    void* out;            // expand: (T, C)
    const void* factor;   // shrink: (A, R, K) or (A, K, R); expand: (A, C, R) or (A, R, C)
    void* v; float* row_scale;  // h or g: planes of (T, R), and the rows' powers of two behind them
    const int* offsets; const int* adapters; const float* scale;
    long long stride_x, stride_out;
    int T, K, R, A, requests;  // K: length of the contraction (shrink), columns (expand)
    int rows_per_item, cols_per_cta;  // (shrink, expand)
    bool chained;         // launched behind a kernel of the same call
    int* status;          // device int32, set non-zero when a bounded wait expires; may be null
};

// The gradients of both factors are one launch: the first `groups` CTAs of a row of the grid are job 0's, U's, with partial
// products (items, K, R); the others job 1's, D's, (items, R, K).
struct OuterJob {
    const void* x; const void* v; const float* row_scale;  // (T, K) and (T, R) operands
    float* part;
    int* item_adapter;  // (items): -1 for an item without rows or adapter
    long long stride_x;
    int K, rows, items;  // columns (0: no such job), rows of an item
};
struct OuterJobs {
    OuterJob job[2];
    int groups;
};

struct Item {
    int first, rows, adapter;  // rows 0: nothing to do; adapter -1: rows without one
};
__host__ __device__ inline int item_count(int T, int requests, int bm) { return (T + bm - 1) / bm + requests + 1; }

// The `w`-th interval of the merged borders (those of tiles of `bm` rows before equal offsets).  All threads of the CTA call it.
template <int THREADS>
__device__ __forceinline__ Item find_item(const LoraParams& p, int w, int bm) {
    const int tiles = (p.T + bm - 1) / bm;
    auto offset = [&](int j) { return min(max(__ldg(p.offsets + j), 0), p.T); };
    int before = 0;  // offsets among the first w borders
    for (int j0 = 0; j0 <= p.requests; j0 += THREADS) {
        const int j = j0 + (int)threadIdx.x;
        before += __syncthreads_count(j <= p.requests && j + min(offset(j) / bm + 1, tiles) < w);
    }
    int i = w - before, j = before;
    Item it = {0, 0, -1};
    const int tile = i < tiles ? i * bm : p.T, off = j <= p.requests ? offset(j) : p.T;
    int next_tile = tile, next_off = off;
    if (i < 0) return it;  // (offsets that go down)
    if (i < tiles && tile <= off) {
        it.first = tile;
        next_tile = i + 1 < tiles ? (i + 1) * bm : p.T;
    } else if (j <= p.requests) {
        it.first = off;
        ++j;
        next_off = j <= p.requests ? offset(j) : p.T;
    } else {
        return it;
    }
    it.rows = min(max(min(next_tile, next_off) - it.first, 0), bm);
    if (it.rows && j >= 1 && j <= p.requests) {
        const int a = __ldg(p.adapters + j - 1);
        it.adapter = a >= 0 && a < p.A ? a : -1;
    }
    return it;
}

// About how many of them have rows.  Long requests add a border inside a tile each: leaving these out started a second wave of
// a few CTAs (5003 rows of 9 requests, 12288 -> 3072, rank 64: 55.2 us, 53.0 with them; 4096 rows of 4 ragged requests, 2048 ->
// 6144: 42.0, 38.0).  Short ones often lie on the tiles' borders, or fill the SMs by themselves: with theirs added, 8192 rows
// of 64 requests of equal length took 73.0 us for 53.1.
inline int live_items(const LoraParams& p, int bm) {
    const int tiles = (p.T + bm - 1) / bm, requests = p.requests < p.T ? p.requests : p.T;
    return tiles >= 4 * requests && requests > 0 ? tiles + requests - 1 : tiles > requests ? tiles : requests;
}

// The kernels of a call form a chain: each is launched while the one before it still runs (programmatic stream
// serialization), does what does not depend on it - finding its item, loading the factor and base - and waits for its end
// before it reads what it wrote, or writes what it may still read.  A kernel that has ended has waited for the one before
// it, so the wait covers all of the chain; its first kernel is launched as usual, after everything before the call.
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster_y, bool chained, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster_y > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = 1;
        at[n].val.clusterDim.y = cluster_y;
        at[n++].val.clusterDim.z = 1;
    }
    if (chained) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    NB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    return NB_OK;
}

inline int sms() {
    const int n = nb_num_sms();
    return n > 0 ? n : 148;
}
inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// The tcgen05 kernels (lora_tc.cu): the same three products for calls with many rows per request.  `p` as for the kernels in
// lora.cu, with rows_per_item set by these (kTcRows for shrink and expand).  NB_ERR_UNSUPPORTED: no tensor map, nothing ran.
constexpr int kTcRows = 128, kTcCols = 256;  // rows of an item (shrink, expand), columns of a CTA (outer)
int tc_shrink(LoraParams p, bool rcontig, int dtype, cudaStream_t s);
int tc_expand(LoraParams p, bool ccontig, int dtype, cudaStream_t s);
int tc_outer(const LoraParams& p, OuterJobs j, int dtype, cudaStream_t s);

}  // namespace lora
}  // namespace nb
