// The products of the batched adapters (lora.cu has the mathematics and the items) on the tcgen05 tensor cores, for calls
// with many rows per request: operands by TMA into 128-byte-swizzled tiles, accumulators in tensor memory, an epilogue
// that overlaps the next tiles.  The products move many bytes per multiplication (rank 64: 32 multiply-adds per byte of x,
// base, out or dy), so what the tensor cores give here is not arithmetic but the absence of it elsewhere: no operand passes
// through registers, and the bytes in flight are the size of the shared-memory ring.  Measured on a B200 (bf16, 9216 rows,
// rank 64, profiled): shrink 3072 -> 64 20.5 us and 9216 -> 64 37 us (2.8 and 4.6 TB/s), expand 64 -> 9216 62 us (5.5 TB/s),
// outer 60 us for both factors (3.9 TB/s): about 8 us of each are its start and its end, the rest its bytes (outer's CTAs are
// of two lengths, and end at different times).
//
// A tensor-memory accumulator is fp32, but each step into it TRUNCATES, the sum and (fp16, whose products have 22 bits) the
// products that it takes: a long chain is biased towards zero (432 steps: 1.4e-5 of the sum; fp32 with rounding 1.7e-6).  The
// long sums (shrink, outer) are therefore taken out of it every 32 to 48 steps and added up in registers, where additions
// round, while the ring keeps the loads coming and a second accumulator takes the next steps.
//
// A tile is loaded whole even where its item has fewer rows: the rows behind belong to other requests (or are filled with
// zeros behind the last row).  They are multiplied along and not stored; where rows are summed (outer) they are set to zero
// in shared memory first.  Every mbarrier wait is bounded; on expiry the CTA records a code in the status word and unwinds.
#include <cooperative_groups.h>
#include <cuda.h>

#include <type_traits>

#include "lora.cuh"

namespace cg = cooperative_groups;

namespace nb {
namespace lora {
namespace {

constexpr int KB = 64;  // values of a 128-byte row of a tile

enum { E_SHRINK = 0x310, E_EXPAND = 0x330, E_OUTER = 0x350 };

// K-major operand (rows along M or N, the 64 values of a 128-byte row along K): 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// MN-major operand (the 64 values of a 128-byte row along M or N, rows along K): 8-row groups 1024 bytes apart along K,
// `half` bytes between 64-wide halves along M or N
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t half) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(half >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
constexpr uint32_t A_MN = 1u << 15, B_MN = 1u << 16;

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(src), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// after a wait that expired: copies in flight land before the CTA's shared memory goes (bounded)
__device__ __forceinline__ void let_copies_land() {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 100000000ull) {}
}
template <typename T>
struct Fmt { static constexpr uint32_t value = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u; };
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(tmap),
                 "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ uint8_t* align1k(unsigned char* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// the planes of h or g as tensor maps
template <typename T>
struct PartMaps {
    CUtensorMap part[Split<T>::PARTS];
};

// ------------------------------------------------------------------------------------------------------------------ shrink
// 128 rows x R over one slice of K; the slices of an item are a cluster whose sums meet in shared memory.
// Warps: TMA producer, MMA issuer, four for the sums.
template <int RP>  // R rounded up to 16, 32, 64 or 128
struct ShrinkTc {
    static constexpr int XB = kTcRows * 128;
    static constexpr int FB = RP <= 64 ? 64 * 128 : 2 * 64 * 128;  // [64 of K][64 r] tiles, or RP rows of 64 of K
    static constexpr int STAGE = XB + FB, ST = RP <= 64 ? 8 : 6;  // 192 KB: one CTA per SM
    static constexpr int LD = RP + 4;  // floats of a row of sums: 16-byte accesses of eight rows on different banks
    static constexpr int PIPE = ST * STAGE, SUMS = kTcRows * LD * 4;
    static constexpr int OFF_BAR = PIPE > SUMS ? PIPE : SUMS;
    static constexpr int BYTES = OFF_BAR + 256 + 1024;
    static constexpr int ACC = RP < 32 ? 32 : RP, COLS = 2 * ACC;  // two accumulators take turns
    static constexpr int THREADS = 192;
    static constexpr int CHAIN = 8;  // steps of 64 of K into an accumulator before it is taken out
};
template <typename T, int RP, bool RCONTIG>
__global__ void __launch_bounds__(192) lora_shrink_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_f,
                                                              const LoraParams p) {
    using S = ShrinkTc<RP>;
    extern __shared__ unsigned char raw[];
    chain_next();
    uint8_t* smem = align1k(raw);
    const uint32_t base = smem_u32(smem), bars = base + S::OFF_BAR;
    auto full = [&](int i) { return bars + 8u * i; };
    auto empty = [&](int i) { return bars + 8u * (S::ST + i); };
    // an accumulator has a chain's sums / may be used again
    auto done = [&](int b) { return bars + 8u * (2 * S::ST + b); };
    auto taken = [&](int b) { return bars + 8u * (2 * S::ST + 2 + b); };
    static_assert(8 * (2 * S::ST + 4) <= 192, "barriers");
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + S::OFF_BAR + 192);
    volatile int* abort_s = reinterpret_cast<volatile int*>(smem + S::OFF_BAR + 200);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (set up while the offsets are on their way)
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_f);
        for (int i = 0; i < S::ST; ++i) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(done(b), 1);
            mbar_init(taken(b), 4);
        }
        *abort_s = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_at), S::COLS);
        tmem_relinquish();
    }
    const Item it = find_item<S::THREADS>(p, blockIdx.x, p.rows_per_item);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    if (it.rows == 0 || it.adapter < 0) {  // every CTA of the cluster
        if (warp == 1) tmem_dealloc(tmem, S::COLS);
        return;
    }
    const int splits = gridDim.y, split = blockIdx.y;
    const int steps = (p.K + KB - 1) / KB, per = (steps + splits - 1) / splits;
    const int step0 = min(split * per, steps), n = min(per, steps - step0);
    // bytes that land per stage (the part of a box outside the tensor arrives as zeros and counts)
    const int fhalves = RP <= 64 ? 1 : 2;

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int s = 0; s < n; ++s) {
                const int st = s % S::ST;
                if (s >= S::ST && !mbar_wait(empty(st), ((s / S::ST) & 1) ^ 1, abort_s, E_SHRINK | 1, 50)) { ok = false; break; }
                const uint32_t x = base + st * S::STAGE, f = x + S::XB;
                const int k0 = (step0 + s) * KB;
                mbar_expect_tx(full(st), S::XB + (RCONTIG ? fhalves * 64 * 128 : p.R * 128));
                tma_load_2d(x, &tm_x, full(st), k0, it.first);
                if constexpr (RCONTIG) {
                    for (int h = 0; h < fhalves; ++h) tma_load_3d(f + h * 64 * 128, &tm_f, full(st), h * 64, k0, it.adapter);
                } else {
                    tma_load_3d(f, &tm_f, full(st), k0, 0, it.adapter);
                }
            }
            if (!ok) let_copies_land();
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc(1u, Fmt<T>::value, Fmt<T>::value, p.R) | (RCONTIG ? B_MN : 0u);
        bool ok = true;
        for (int s = 0; s < n && ok; ++s) {
            const int st = s % S::ST;
            if (!mbar_wait_warp(full(st), (s / S::ST) & 1, abort_s, E_SHRINK | 2)) { ok = false; break; }
            const int chain = s / S::CHAIN, b = chain & 1;
            if (chain >= 2 && s % S::CHAIN == 0 && !mbar_wait_warp(taken(b), ((chain >> 1) - 1) & 1, abort_s, E_SHRINK | 4)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint64_t a = desc_k(base + st * S::STAGE);
                const uint64_t f = RCONTIG ? desc_mn(base + st * S::STAGE + S::XB, 64 * 128) : desc_k(base + st * S::STAGE + S::XB);
                const int k16 = min(4, (p.K - (step0 + s) * KB + 15) / 16);
                for (int k = 0; k < k16; ++k) mma_f16(tmem + b * S::ACC, a + k * 2, f + k * (RCONTIG ? 16 * 128 >> 4 : 2), idesc, (s % S::CHAIN || k) ? 1u : 0u);
                tc_commit(empty(st));
                if (s == n - 1 || s % S::CHAIN == S::CHAIN - 1) tc_commit(done(b));
            }
            __syncwarp();
        }
    }
    const float scale = p.scale ? __ldg(p.scale + it.adapter) : 1.f;
    float* sums = reinterpret_cast<float*>(smem);
    if (warp >= 2) {
        bool ok = true;
        const int row = (warp & 3) * 32 + lane;
        float total[RP] = {};
        for (int s = 0, chain = 0; s < n && ok; s += S::CHAIN, ++chain) {
            ok = mbar_wait_warp(done(chain & 1), (chain >> 1) & 1, abort_s, E_SHRINK | 3);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < RP; c += 32) {
                float v[32];
                tmem_ld32(tmem + ((warp & 3) * 32 << 16) + (chain & 1) * S::ACC + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < (RP < 32 ? RP : 32); ++i) total[c + i] += v[i];
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(taken(chain & 1));
            __syncwarp();
        }
        if (ok) {
#pragma unroll
            for (int i = 0; i < RP; i += 4)
                *reinterpret_cast<float4*>(sums + row * S::LD + i) = make_float4(total[i], total[i + 1], total[i + 2], total[i + 3]);
        }
    }
    __syncthreads();
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync();
    // LANES neighbours have a row, each four of its ranks; the slices' sums in order, all the loads of a value on their way together
    constexpr int LANES = RP / 4, TEAMS = S::THREADS / LANES, PARTS = Split<T>::PARTS;
    for (int r0 = split * TEAMS; r0 < it.rows; r0 += splits * TEAMS) {
        const int row = r0 + (int)threadIdx.x / LANES, r = (int)threadIdx.x % LANES * 4;
        const bool on = row < it.rows && r < p.R;
        float4 u[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (on && q < splits) u[q] = *reinterpret_cast<const float4*>((splits > 1 ? cluster.map_shared_rank(sums, q) : sums) + row * S::LD + r);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (on && q < splits) { v.x += u[q].x; v.y += u[q].y; v.z += u[q].z; v.w += u[q].w; }
        v.x *= scale; v.y *= scale; v.z *= scale; v.w *= scale;
        if constexpr (Split<T>::SCALED) {
            float big = fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const int e = row_exponent(big);
            const float down = exp2_of(-e);
            v.x *= down; v.y *= down; v.z *= down; v.w *= down;
            if (r == 0 && on) p.row_scale[it.first + row] = exp2_of(e);
        }
        if (!on) continue;
        uint32_t xy[PARTS], zw[PARTS];
        split_pair<T>(v.x, v.y, xy);
        split_pair<T>(v.z, v.w, zw);
#pragma unroll
        for (int k = 0; k < PARTS; ++k)
            *reinterpret_cast<uint2*>(static_cast<char*>(p.v) + k * plane_bytes(p.T, p.R) + ((long long)(it.first + row) * p.R + r) * 2) = make_uint2(xy[k], zw[k]);
    }
    if (splits > 1) cluster.sync();
    else __syncthreads();
    if (*abort_s) let_copies_land();
    if (threadIdx.x == 0 && *abort_s && p.status) atomicCAS(p.status, 0, *abort_s);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, S::COLS);
    }
}

// ------------------------------------------------------------------------------------------------------------------ expand
// out[128 rows, columns col0 .. col1) = base + v G^T, 64 columns at a time.  The parts of the item's v stay in shared
// memory; a ring of SLOTS 16 KB tiles carries base in and out back: TMA load, tensor-memory result added in place, TMA
// store (straight from registers where the item has fewer than 128 rows).  Warps: TMA producer, MMA issuer, eight that add
// (a lane has a row, a warp half of a tile's columns), one that stores.  All of them take every tile, in order: a barrier of
// the ring is then never more than one phase ahead of anybody who waits on it.
template <typename T, int RP>
struct ExpandTc {
    static constexpr int HALVES = RP <= 64 ? 1 : 2, PARTS = Split<T>::PARTS;
    static constexpr int VB = HALVES * kTcRows * 128;   // a part of v
    // up to rank 64 two CTAs share an SM, so that one starts and drains under the other's tiles
    static constexpr int PER_SM = RP <= 64 ? 2 : 1;
    static constexpr int GB = HALVES * 64 * 128, GST = RP <= 64 ? 2 : 3;
    static constexpr int SLOT = kTcRows * 128, SLOTS = RP <= 64 ? 3 : 5;
    static constexpr int OFF_G = PARTS * VB, OFF_S = OFF_G + GST * GB, OFF_BAR = OFF_S + SLOTS * SLOT;
    static constexpr int BYTES = OFF_BAR + 256;  // (no room to align it by hand: 114944 bytes at rank 64, 115712 fit twice)
    static constexpr int THREADS = 352;
};
extern __shared__ __align__(1024) unsigned char expand_smem[];
template <typename T, int RP, bool CCONTIG>
__global__ void __launch_bounds__(352) lora_expand_tc_kernel(const __grid_constant__ PartMaps<T> tm_v, const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_base,
                                                              const __grid_constant__ CUtensorMap tm_out, const LoraParams p) {
    using S = ExpandTc<T, RP>;
    const Item it = find_item<S::THREADS>(p, blockIdx.y, p.rows_per_item);
    if (it.rows == 0) return;
    const int col0 = blockIdx.x * p.cols_per_cta, col1 = min(col0 + p.cols_per_cta, p.K);
    const T* in = static_cast<const T*>(p.x);
    T* out = static_cast<T*>(p.out);
    if (it.adapter < 0) {  // base alone (zeros without one)
        chain_wait();
        if (in == out) return;
        const int n = (col1 - col0) / 8;
        for (int e = threadIdx.x; e < it.rows * n; e += S::THREADS) {
            const int row = e / n, c = col0 + (e - row * n) * 8;
            const uint4 v = in ? *reinterpret_cast<const uint4*>(in + (it.first + row) * p.stride_x + c) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + (it.first + row) * p.stride_out + c) = v;
        }
        return;
    }
    unsigned char* smem = expand_smem;
    const uint32_t sb = smem_u32(smem), bars = sb + S::OFF_BAR;
    auto bar = [&](int i) { return bars + 8u * i; };
    enum { V = 0, GF = 1, GE = GF + S::GST, DF = GE + S::GST, DE = DF + 2, LF = DE + 2, LE = LF + S::SLOTS, WF = LE + S::SLOTS, COUNT = WF + S::SLOTS };
    // V, G: operands landed / free; D: accumulator done / read; L: a slot's base landed / the slot free; W: its result written
    static_assert(COUNT * 8 <= 224, "barriers");
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + S::OFF_BAR + 224);
    volatile int* abort_s = reinterpret_cast<volatile int*>(smem + S::OFF_BAR + 232);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(bar(V), 1);
        for (int i = 0; i < S::GST; ++i) { mbar_init(bar(GF + i), 1); mbar_init(bar(GE + i), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(DF + i), 1); mbar_init(bar(DE + i), 8); }
        for (int i = 0; i < S::SLOTS; ++i) { mbar_init(bar(LF + i), 1); mbar_init(bar(LE + i), 1); mbar_init(bar(WF + i), 8); }
        *abort_s = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_at), 128);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    const int tiles = (col1 - col0 + 63) / 64;
    const bool has_base = in != nullptr;

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int i = 0; i < tiles; ++i) {
                const int c = col0 + i * 64, gs = i % S::GST, ls = i % S::SLOTS;
                if (i >= S::GST && !mbar_wait(bar(GE + gs), ((i / S::GST) & 1) ^ 1, abort_s, E_EXPAND | 1, 50)) { ok = false; break; }
                const uint32_t g = sb + S::OFF_G + gs * S::GB;
                if constexpr (CCONTIG) {  // R rows of 64 columns
                    mbar_expect_tx(bar(GF + gs), p.R * 128);
                    tma_load_3d(g, &tm_g, bar(GF + gs), c, 0, it.adapter);
                } else {  // 64 rows (columns of out) of R
                    mbar_expect_tx(bar(GF + gs), S::GB);
                    for (int h = 0; h < S::HALVES; ++h) tma_load_3d(g + h * 64 * 128, &tm_g, bar(GF + gs), h * 64, c, it.adapter);
                }
                if (has_base) {
                    if (i >= S::SLOTS && !mbar_wait(bar(LE + ls), ((i / S::SLOTS) & 1) ^ 1, abort_s, E_EXPAND | 2, 50)) { ok = false; break; }
                    mbar_expect_tx(bar(LF + ls), S::SLOT);
                    tma_load_2d(sb + S::OFF_S + ls * S::SLOT, &tm_base, bar(LF + ls), c, it.first);
                }
                if (i == min(S::GST, tiles) - 1) {  // the ring is filled as far as it goes without the kernel before this one
                    chain_wait();
                    mbar_expect_tx(bar(V), S::PARTS * S::VB);
                    for (int h = 0; h < S::HALVES; ++h)
                        for (int v = 0; v < S::PARTS; ++v) tma_load_2d(sb + v * S::VB + h * kTcRows * 128, &tm_v.part[v], bar(V), h * 64, it.first);
                }
            }
            if (!ok) let_copies_land();
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc(1u, Fmt<T>::value, Fmt<T>::value, 64) | (CCONTIG ? B_MN : 0u);
        const int k16 = p.R / 16;
        bool ok = mbar_wait_warp(bar(V), 0, abort_s, E_EXPAND | 3);
        for (int i = 0; i < tiles && ok; ++i) {
            const int gs = i % S::GST, d = i & 1;
            if (!mbar_wait_warp(bar(GF + gs), (i / S::GST) & 1, abort_s, E_EXPAND | 4)) { ok = false; break; }
            if (i >= 2 && !mbar_wait_warp(bar(DE + d), ((i >> 1) & 1) ^ 1, abort_s, E_EXPAND | 5)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint32_t g = sb + S::OFF_G + gs * S::GB;
                for (int v = 0; v < S::PARTS; ++v)
                    for (int k = 0; k < k16; ++k) {
                        const uint64_t a = desc_k(sb + v * S::VB + (k >> 2) * kTcRows * 128) + (k & 3) * 2;
                        const uint64_t b = CCONTIG ? desc_mn(g + k * 16 * 128, 64 * 128) : desc_k(g + (k >> 2) * 64 * 128) + (k & 3) * 2;
                        mma_f16(tmem + d * 64, a, b, idesc, (v || k) ? 1u : 0u);
                    }
                tc_commit(bar(GE + gs));
                tc_commit(bar(DF + d));
            }
            __syncwarp();
        }
    } else if (warp < 10) {
        const int q = warp & 3, half = (warp - 2) >> 2, row = q * 32 + lane;
        const bool whole = it.rows == kTcRows;
        float power = 1.f;  // of this lane's row
        if constexpr (Split<T>::SCALED) {
            chain_wait();
            if (row < it.rows) power = *const_cast<const volatile float*>(p.row_scale + it.first + row);
        }
        for (int i = 0; i < tiles; ++i) {
            const int ls = i % S::SLOTS, d = i & 1, c = col0 + i * 64 + half * 32;
            const uint32_t line = sb + S::OFF_S + ls * S::SLOT + row * 128;
            if (!mbar_wait_warp(bar(DF + d), (i >> 1) & 1, abort_s, E_EXPAND | 6)) break;
            tc_fence_after();
            float v[32];
            tmem_ld32(tmem + (q * 32 << 16) + d * 64 + half * 32, v);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(DE + d));
            __syncwarp();
            if (has_base) {
                if (!mbar_wait_warp(bar(LF + ls), (i / S::SLOTS) & 1, abort_s, E_EXPAND | 7)) break;
            } else if (i >= S::SLOTS) {  // nobody loads into the slot, but its last store has to have read it
                if (!mbar_wait_warp(bar(LE + ls), ((i / S::SLOTS) & 1) ^ 1, abort_s, E_EXPAND | 8)) break;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t at = line + (((half * 4 + j) ^ (row & 7)) << 4);
                const float* f = v + j * 8;
                uint4 o;
                if (has_base) {
                    uint4 b;
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "r"(at) : "memory");
                    const float2 b0 = unpack2<T>(b.x), b1 = unpack2<T>(b.y), b2 = unpack2<T>(b.z), b3 = unpack2<T>(b.w);
                    const auto add = [&](float v0, float v1, float2 u) { return pack2<T>(fmaf(v0, power, u.x), fmaf(v1, power, u.y)); };
                    o = make_uint4(add(f[0], f[1], b0), add(f[2], f[3], b1), add(f[4], f[5], b2), add(f[6], f[7], b3));
                } else {
                    const auto one = [&](float v0, float v1) { return pack2<T>(v0 * power, v1 * power); };
                    o = make_uint4(one(f[0], f[1]), one(f[2], f[3]), one(f[4], f[5]), one(f[6], f[7]));
                }
                if (whole)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w) : "memory");
                else if (row < it.rows && c + j * 8 < col1)
                    *reinterpret_cast<uint4*>(out + (it.first + row) * p.stride_out + c + j * 8) = o;
            }
            fence_proxy_async_smem();  // what was written is stored, and what was read is loaded over, by the async proxy
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(WF + ls));
            __syncwarp();
        }
    } else if (lane == 0) {
        for (int i = 0; i < tiles; ++i) {
            const int ls = i % S::SLOTS;
            if (!mbar_wait(bar(WF + ls), (i / S::SLOTS) & 1, abort_s, E_EXPAND | 9, 50)) break;
            if (it.rows == kTcRows) {
                tma_store_2d(&tm_out, sb + S::OFF_S + ls * S::SLOT, col0 + i * 64, it.first);
                bulk_commit();
                bulk_wait_read<0>();
            }
            mbar_arrive(bar(LE + ls));
        }
        bulk_wait_all();
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_s) let_copies_land();
    if (threadIdx.x == 0 && *abort_s && p.status) atomicCAS(p.status, 0, *abort_s);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 128);
    }
}

// ------------------------------------------------------------------------------------------------------------------- outer
// part[item][r, k] (job 1; [k, r] for job 0) = sum over the item's rows of v[t, r] X[t, k], 256 columns of X per CTA
// (two accumulators of 128: v comes from the L2 cache once for both, 16 KB beside 32 KB of X at rank 64; with 128
// columns the cache delivered as much of it as HBM of X).  Both operands run along the rows (MN-major), so they are used
// as they lie.  Warps: TMA producer, MMA issuer, eight for the sums (four for each accumulator); where the rows have powers of
// two, these bring the rows of v to the item's power in shared memory before they are multiplied.
template <typename T, int RP>
struct OuterTc {
    static constexpr int HALVES = RP <= 64 ? 1 : 2, PARTS = Split<T>::PARTS;
    // rows of a stage: 64, or 32 where a stage of 64 is so large (80 KB) that two alone would fit
    static constexpr int ROWS = PARTS * HALVES > 4 ? 32 : 64;
    static constexpr int TILE = ROWS * 128;  // of 64 values
    static constexpr int STAGE = (4 + PARTS * HALVES) * TILE, ST = ROWS == 32 ? 5 : RP <= 64 ? 4 : 3;
    static constexpr int OFF_BAR = ST * STAGE;
    static constexpr int BYTES = OFF_BAR + 256 + 1024;
    // Up to rank 64 the parts of v are one operand, 64 columns each: X is read from shared memory once for all (one at a time,
    // three parts of rank 64 read 144 KB for a stage of 56), and the small parts do not meet the truncation of the large.
    static constexpr bool WIDE = RP <= 64;
    static constexpr int ACC = WIDE ? PARTS * 64 : RP, COLS = 2 * ACC <= 256 ? 256 : 512;  // tensor-memory columns: two accumulators
    static constexpr int THREADS = 320;
    static constexpr int CHAIN = (WIDE ? 512 : 256) / ROWS;  // stages into the accumulators before they are taken out
};
template <typename T>
struct OuterMaps {
    CUtensorMap x[2];  // of the two jobs
    PartMaps<T> v[2];
};
template <typename T, int RP>
__global__ void __launch_bounds__(320) lora_outer_tc_kernel(const __grid_constant__ OuterMaps<T> maps, const LoraParams p,
                                                            const __grid_constant__ OuterJobs jobs) {
    using S = OuterTc<T, RP>;
    constexpr bool SCALED = Split<T>::SCALED;
    const bool krows = (int)blockIdx.x < jobs.groups;
    const int which = krows ? 0 : 1, K = jobs.job[which].K;
    const CUtensorMap& tm_x = maps.x[which];
    const PartMaps<T>& tm_v = maps.v[which];
    extern __shared__ unsigned char raw[];
    chain_next();
    uint8_t* smem = align1k(raw);
    const uint32_t sb = smem_u32(smem), bars = sb + S::OFF_BAR;
    auto full = [&](int i) { return bars + 8u * i; };
    auto empty = [&](int i) { return bars + 8u * (S::ST + i); };
    auto level = [&](int i) { return bars + 8u * (2 * S::ST + i); };  // a slot's rows of v have the item's power
    const uint32_t done = bars + 8u * (3 * S::ST), taken = done + 8;  // (as in shrink)
    static_assert(8 * (3 * S::ST + 2) <= 192, "barriers");
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + S::OFF_BAR + 192);
    volatile int* abort_s = reinterpret_cast<volatile int*>(smem + S::OFF_BAR + 200);
    int* tops = reinterpret_cast<int*>(smem + S::OFF_BAR + 208);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (set up while the offsets are on their way)
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_x);
        for (int k = 0; k < S::PARTS; ++k) tma_prefetch_desc(&tm_v.part[k]);
        for (int i = 0; i < S::ST; ++i) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), 1);
            mbar_init(level(i), 8);
        }
        mbar_init(done, 1);
        mbar_init(taken, 8);
        *abort_s = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_at), S::COLS);
        tmem_relinquish();
    }
    // last items first: their rows are the ones that the kernel before this one read last and left in the L2 cache
    const int w = jobs.job[which].items - 1 - (int)blockIdx.y;
    const Item it = find_item<S::THREADS>(p, w, jobs.job[which].rows);
    chain_wait();
    if (blockIdx.x == (krows ? 0 : jobs.groups) && threadIdx.x == 0 && w >= 0) jobs.job[which].item_adapter[w] = it.rows ? it.adapter : -1;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;
    if (w < 0 || it.rows == 0 || it.adapter < 0) {  // (w: the other job has more items)
        if (warp == 1) tmem_dealloc(tmem, S::COLS);
        return;
    }
    const int c0 = (blockIdx.x - (krows ? 0 : jobs.groups)) * kTcCols, n = (it.rows + S::ROWS - 1) / S::ROWS;
    const int quarters = min(4, (K - c0 + 63) / 64);  // tiles of 64 columns that exist

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int s = 0; s < n; ++s) {
                const int st = s % S::ST, t0 = it.first + s * S::ROWS;
                if (s >= S::ST && !mbar_wait(empty(st), ((s / S::ST) & 1) ^ 1, abort_s, E_OUTER | 1, 50)) { ok = false; break; }
                const uint32_t at = sb + st * S::STAGE;
                mbar_expect_tx(full(st), (quarters + S::PARTS * S::HALVES) * S::TILE);
                for (int q = 0; q < quarters; ++q) tma_load_2d(at + q * S::TILE, &tm_x, full(st), c0 + q * 64, t0);
                for (int v = 0; v < S::PARTS; ++v)
                    for (int h = 0; h < S::HALVES; ++h) tma_load_2d(at + (4 + v * S::HALVES + h) * S::TILE, &tm_v.part[v], full(st), h * 64, t0);
            }
            if (!ok) let_copies_land();
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc(1u, Fmt<T>::value, Fmt<T>::value, S::WIDE ? S::ACC : p.R) | A_MN | B_MN;
        bool ok = true;
        for (int s = 0; s < n && ok; ++s) {
            const int st = s % S::ST, rows = min(S::ROWS, it.rows - s * S::ROWS), k16 = (rows + 15) / 16;
            const uint32_t at = sb + st * S::STAGE;
            if (!mbar_wait_warp(full(st), (s / S::ST) & 1, abort_s, E_OUTER | 2)) { ok = false; break; }
            if (rows < k16 * 16) {  // rows behind the item's last one: zeros in every tile
                for (int tile = 0; tile < 4 + S::PARTS * S::HALVES; ++tile)
                    for (int e = rows * 8 + lane; e < k16 * 16 * 8; e += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at + tile * S::TILE + e * 16), "r"(0) : "memory");
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (s && s % S::CHAIN == 0 && !mbar_wait_warp(taken, (s / S::CHAIN - 1) & 1, abort_s, E_OUTER | 6)) { ok = false; break; }
            if (SCALED && !mbar_wait_warp(level(st), (s / S::ST) & 1, abort_s, E_OUTER | 4)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
                for (int k = 0; k < k16; ++k)
                    for (int h = 0; 2 * h < quarters; ++h) {
                        const uint64_t a = desc_mn(at + 2 * h * S::TILE + k * 16 * 128, S::TILE);
                        for (int v = 0; v < (S::WIDE ? 1 : S::PARTS); ++v)
                            mma_f16(tmem + h * S::ACC, a, desc_mn(at + (4 + v * S::HALVES) * S::TILE + k * 16 * 128, S::TILE), idesc, (s % S::CHAIN || k || v) ? 1u : 0u);
                    }
                tc_commit(empty(st));
                if (s == n - 1 || s % S::CHAIN == S::CHAIN - 1) tc_commit(done);
            }
            __syncwarp();
        }
    } else {
        const int q = warp & 3, h = (warp - 2) >> 2;
        float* part = jobs.job[which].part + (long long)w * p.R * K;
        const float* powers = jobs.job[which].row_scale + it.first;
        // four threads have a row of a slot, each two of its eight 16-byte pieces
        const int t = threadIdx.x - 64, row = t >> 2;
        int top = 0;
        float next = 1.f, total[RP] = {};
        bool ok = true;
        if constexpr (SCALED) {
            static_assert(S::ROWS == 64, "64 rows, 256 threads");
            top = -126;
#pragma unroll 4
            for (int r = t; r < it.rows; r += 256) top = max(top, (int)(__float_as_uint(powers[r]) >> 23) - 127);
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) tops[warp - 2] = top;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
            if (row < it.rows) next = powers[row];
        }
        for (int s = 0; s < n; ++s) {
            if constexpr (SCALED) {
                const int st = s % S::ST;
                float a, b;
                row_ratio(next, top, a, b);
                if ((s + 1) * S::ROWS + row < it.rows) next = powers[(s + 1) * S::ROWS + row];
                if (!mbar_wait_warp(full(st), (s / S::ST) & 1, abort_s, E_OUTER | 5)) { ok = false; break; }
                if (s * S::ROWS + row < it.rows && a * b < 1.f) {
                    const __half2 a2 = __float2half2_rn(a), b2 = __float2half2_rn(b);
                    const uint32_t at = sb + st * S::STAGE + 4 * S::TILE + row * 128 + (t & 3) * 32;
                    for (int tile = 0; tile < S::PARTS * S::HALVES; ++tile)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t v[4];
                            const uint32_t to = at + tile * S::TILE + c * 16;
                            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(to) : "memory");
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                __half2 x2 = *reinterpret_cast<__half2*>(&v[j]);
                                x2 = __hmul2(__hmul2(x2, a2), b2);
                                v[j] = *reinterpret_cast<uint32_t*>(&x2);
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                        }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(level(st));
                __syncwarp();
            }
            if (s != n - 1 && s % S::CHAIN != S::CHAIN - 1) continue;
            if (!mbar_wait_warp(done, (s / S::CHAIN) & 1, abort_s, E_OUTER | 3)) { ok = false; break; }
            tc_fence_after();
            if (2 * h < quarters) {
#pragma unroll
                for (int part = S::WIDE ? S::PARTS - 1 : 0; part >= 0; --part)  // the smallest first
#pragma unroll
                    for (int c = 0; c < RP; c += 32) {
                        float v[32];
                        tmem_ld32(tmem + (q * 32 << 16) + h * S::ACC + part * 64 + c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < (RP < 32 ? RP : 32); ++i) total[c + i] += v[i];
                    }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(taken);
            __syncwarp();
        }
        const int k = c0 + h * 128 + q * 32 + lane;
        if (ok && 2 * h < quarters && k < K) {
            if constexpr (SCALED) {
                const float up = exp2_of(top);
#pragma unroll
                for (int i = 0; i < RP; ++i) total[i] *= up;
            }
            if (krows) {
                float* to = part + (long long)k * p.R;
#pragma unroll
                for (int i = 0; i < RP; i += 8)
                    if (i < p.R)
                        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to + i), "f"(total[i]), "f"(total[i + 1]),
                                     "f"(total[i + 2]), "f"(total[i + 3]), "f"(total[i + 4]), "f"(total[i + 5]), "f"(total[i + 6]), "f"(total[i + 7]) : "memory");
            } else {
#pragma unroll
                for (int i = 0; i < RP; ++i)
                    if (i < p.R) part[(long long)i * K + k] = total[i];
            }
        }
    }
    __syncthreads();
    if (*abort_s) let_copies_land();
    if (threadIdx.x == 0 && *abort_s && p.status) atomicCAS(p.status, 0, *abort_s);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, S::COLS);
    }
}

// --------------------------------------------------------------------------------------------------------------- launchers
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult res;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiledFn>(sym)
                   : nullptr;
    }();
    return fn;
}
// `depth` matrices (0: one, as a 2-D map) of (rows, cols) 16-bit values one behind the other, `stride` elements between rows;
// boxes of 64 columns by `box_rows` rows of one matrix, zeros outside it
template <typename T>
bool make_map(CUtensorMap* m, const void* base, long long rows, long long cols, long long stride, int box_rows, int depth = 0) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
    const cuuint64_t strides[2] = {(cuuint64_t)stride * 2, (cuuint64_t)(stride * rows) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    return fn(m, std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, depth > 0 ? 3 : 2,
              const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
bool make_part_maps(PartMaps<T>* m, const void* v, const LoraParams& p, int box_rows) {
    bool ok = true;
    for (int k = 0; k < Split<T>::PARTS; ++k) ok = ok && make_map<T>(&m->part[k], static_cast<const char*>(v) + k * plane_bytes(p.T, p.R), p.T, p.R, p.R, box_rows);
    return ok;
}

template <typename T, int RP, bool RCONTIG>
int shrink(LoraParams p, cudaStream_t s) {
    using S = ShrinkTc<RP>;
    p.rows_per_item = kTcRows;
    auto* kernel = lora_shrink_tc_kernel<T, RP, RCONTIG>;
    // (before the tensor maps: it makes the device's context current in a thread that has not used it yet)
    NB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
    CUtensorMap x, f;
    const bool ok = make_map<T>(&x, p.x, p.T, p.K, p.stride_x, kTcRows) &&
                    (RCONTIG ? make_map<T>(&f, p.factor, p.K, p.R, p.R, KB, p.A) : make_map<T>(&f, p.factor, p.R, p.K, p.K, p.R, p.A));
    if (!ok) return NB_ERR_UNSUPPORTED;
    const int items = item_count(p.T, p.requests, kTcRows), live = live_items(p, kTcRows);
    // CTAs of an item: as many as fit the SMs in one wave of one each, up to eight (a portable cluster), each with at least four
    // steps of 64 of K
    int splits = sms() / live;
    if (splits > ceil_div(p.K, 4 * KB)) splits = ceil_div(p.K, 4 * KB);
    if (splits > 8) splits = 8;
    if (splits < 1) splits = 1;
    return launch(kernel, dim3(items, splits), S::THREADS, S::BYTES, splits, p.chained, s, x, f, p);
}
template <typename T, int RP, bool CCONTIG>
int expand(LoraParams p, cudaStream_t s) {
    using S = ExpandTc<T, RP>;
    p.rows_per_item = kTcRows;
    auto* kernel = lora_expand_tc_kernel<T, RP, CCONTIG>;
    NB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
    PartMaps<T> v;
    CUtensorMap g, base, out;
    bool ok = make_part_maps<T>(&v, p.v, p, kTcRows) && make_map<T>(&out, p.out, p.T, p.K, p.stride_out, kTcRows) &&
              (CCONTIG ? make_map<T>(&g, p.factor, p.R, p.K, p.K, p.R, p.A) : make_map<T>(&g, p.factor, p.K, p.R, p.R, 64, p.A));
    if (ok && p.x) ok = make_map<T>(&base, p.x, p.T, p.K, p.stride_x, kTcRows);
    else base = out;
    if (!ok) return NB_ERR_UNSUPPORTED;
    const int items = item_count(p.T, p.requests, kTcRows), live = live_items(p, kTcRows);
    // columns of a CTA: the cut of a row into `cuts` pieces that is done soonest, a CTA's cost being its tiles (0.7 us of an
    // SM's share of HBM each) and about three microseconds to start and to load the item's v, waves of the CTAs that
    // are resident together taking turns
    const int tiles = ceil_div(p.K, 64), slots = S::PER_SM * sms();
    int per = tiles;
    float best = 1e30f;
    for (int cuts = 1; cuts <= 64 && cuts <= tiles; ++cuts) {
        const int t = ceil_div(tiles, cuts);
        const float cost = (float)ceil_div((long long)live * ceil_div(tiles, t), slots) * (0.7f * S::PER_SM * t + 3.f);
        if (cost < best) best = cost, per = t;
    }
    p.cols_per_cta = per * 64;
    return launch(kernel, dim3(ceil_div(tiles, per), items), S::THREADS, S::BYTES, 1, p.chained, s, v, g, base, out, p);
}
template <typename T, int RP>
int outer(const LoraParams& p, OuterJobs j, cudaStream_t s) {
    using S = OuterTc<T, RP>;
    auto* kernel = lora_outer_tc_kernel<T, RP>;
    NB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
    OuterMaps<T> m;
    int groups = 0;
    for (int i = 0; i < 2; ++i) {
        const OuterJob& o = j.job[j.job[i].K ? i : 1 - i];  // (a job that is not there has no CTAs; its maps are the other's)
        if (!(make_map<T>(&m.x[i], o.x, p.T, o.K, o.stride_x, S::ROWS) && make_part_maps<T>(&m.v[i], o.v, p, S::ROWS))) return NB_ERR_UNSUPPORTED;
        groups += ceil_div(j.job[i].K, kTcCols);
    }
    j.groups = ceil_div(j.job[0].K, kTcCols);
    const int items = j.job[0].items > j.job[1].items ? j.job[0].items : j.job[1].items;
    return launch(kernel, dim3(groups, items), S::THREADS, S::BYTES, 1, p.chained, s, m, p, j);
}

#define NB_LORA_RP(CALL)                         \
    if (p.R <= 16) return CALL(16);              \
    if (p.R <= 32) return CALL(32);              \
    if (p.R <= 64) return CALL(64);              \
    return CALL(128)

template <typename T>
int shrink_t(const LoraParams& p, bool rcontig, cudaStream_t s) {
#define NB_CALL(RP) (rcontig ? shrink<T, RP, true>(p, s) : shrink<T, RP, false>(p, s))
    NB_LORA_RP(NB_CALL);
#undef NB_CALL
}
template <typename T>
int expand_t(const LoraParams& p, bool ccontig, cudaStream_t s) {
#define NB_CALL(RP) (ccontig ? expand<T, RP, true>(p, s) : expand<T, RP, false>(p, s))
    NB_LORA_RP(NB_CALL);
#undef NB_CALL
}
template <typename T>
int outer_t(const LoraParams& p, const OuterJobs& j, cudaStream_t s) {
#define NB_CALL(RP) (outer<T, RP>(p, j, s))
    NB_LORA_RP(NB_CALL);
#undef NB_CALL
}

}  // namespace

int tc_shrink(LoraParams p, bool rcontig, int dtype, cudaStream_t s) {
    return dtype == NB_DTYPE_BF16 ? shrink_t<__nv_bfloat16>(p, rcontig, s) : shrink_t<__half>(p, rcontig, s);
}
int tc_expand(LoraParams p, bool ccontig, int dtype, cudaStream_t s) {
    return dtype == NB_DTYPE_BF16 ? expand_t<__nv_bfloat16>(p, ccontig, s) : expand_t<__half>(p, ccontig, s);
}
int tc_outer(const LoraParams& p, OuterJobs j, int dtype, cudaStream_t s) {
    return dtype == NB_DTYPE_BF16 ? outer_t<__nv_bfloat16>(p, j, s) : outer_t<__half>(p, j, s);
}

}  // namespace lora
}  // namespace nb
