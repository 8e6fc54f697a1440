// What the kernels of the batched adapters share: their parameters and how the work is cut into items.
#pragma once

#include "nb_common.cuh"

namespace nb {
namespace lora {

struct LoraParams {
    const void* x;        // shrink: (T, K) operand; expand: base (T, C) or null; outer: (T, K) operand
    void* out;            // expand: (T, C)
    const void* factor;   // shrink: (A, R, K) or (A, K, R); expand: (A, C, R) or (A, R, C)
    void* hi; void* lo;   // (T, R) each
    float* part;          // outer: (items, R, K) or (items, K, R)
    int* item_adapter;    // outer: (items)
    const int* offsets; const int* adapters; const float* scale;
    long long stride_x, stride_out;
    int T, K, R, A, requests;  // K: length of the contraction (shrink), columns (expand, outer)
    int rows_per_item, cols_per_cta;
    int* status;          // device int32, set non-zero when a bounded wait expires; may be null
};

struct Item {
    int first, rows, adapter;  // rows 0: nothing to do; adapter -1: rows without one
};
__host__ __device__ inline int item_count(int T, int requests, int bm) { return (T + bm - 1) / bm + requests + 1; }

// The `w`-th interval of the merged borders (tile borders before equal offsets).  All threads of the CTA call it.
template <int THREADS>
__device__ __forceinline__ Item find_item(const LoraParams& p, int w) {
    const int bm = p.rows_per_item, tiles = (p.T + bm - 1) / bm;
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

inline int sms() {
    const int n = nb_num_sms();
    return n > 0 ? n : 148;
}
inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// The tcgen05 kernels (lora_tc.cu): the same three products for calls with many rows per request.  `p` as for the kernels in
// lora.cu, with rows_per_item set by these (kTcRows for shrink and expand).  NB_ERR_UNSUPPORTED: no tensor map, nothing ran.
constexpr int kTcRows = 128;
int tc_shrink(LoraParams p, bool rcontig, int dtype, cudaStream_t s);
int tc_expand(LoraParams p, bool ccontig, int dtype, cudaStream_t s);
int tc_outer(const LoraParams& p, bool krows, int dtype, cudaStream_t s);

}  // namespace lora
}  // namespace nb
