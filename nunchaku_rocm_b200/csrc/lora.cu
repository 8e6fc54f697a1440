// Low-rank adapters of many requests at once beside a shared projection, forward and backward.
//
// Rows [offsets[i], offsets[i+1]) of x belong to request i, which uses adapter a = adapters[i] (outside 0 .. A-1: none):
//
//     h   = x D_a^T               D (A, R, K)      (shrink)
//     out = base + s_a h U_a^T    U (A, N, R)      (expand)
//     g   = s_a dy U_a                             (shrink)
//     dx  = g D_a                                  (expand)
//     dD_a = sum of g^T x,  dU_a = sum of s_a dy^T h   over the rows of all requests of a   (outer, then join)
//
// Three kernels, each with either order of its factor's elements, cover the six products.  Work is cut into ITEMS: the
// intervals between neighbouring borders, borders being the requests' offsets and every BM-th row.  An item therefore has one
// adapter and at most BM rows, there are at most T / BM + requests + 2 of them however ragged the requests are (so the
// grid is known without reading the offsets on the host), every row is in exactly one, and a CTA finds its item with one
// pass over the offsets: border j of the offsets has floor(offset / BM) + 1 tile borders before it.
//
// h and g are sums in fp32.  Where they are operands again they are held as several 16-bit numbers that add up to them: three
// in bf16 (all 24 bits), two in fp16 after a power of two per row (22 bits; Split, lora.cuh).  One rounding alone would add an
// error as large as that of the output itself.  It multiplies the matrix instructions of the second products, which move more
// bytes than they compute.
//
// Bound: HBM for ranks up to 64 or so (R multiply-adds per byte of x, base or out); for a few rows the latency of two
// dependent kernels, 24 single rows of 24 requests, 3072 -> 18432, rank 16: 13.0 us back to back in a graph.  The forward
// pass of so few rows is one kernel therefore (9.8 us; the floor by bytes is 2).
#include <cooperative_groups.h>

#include "lora.cuh"

namespace cg = cooperative_groups;

namespace nb {
namespace lora {
namespace {

constexpr int kThreads = 128;
constexpr int kRows = 64;  // rows of an item (shrink, expand)

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// 16 bytes to shared memory, or 16 zero bytes (nothing is read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ------------------------------------------------------------------------------------------------------------------ shrink
// v[t, r] = s_a sum_k X[t, k] F_a[r, k], written in parts.  A CTA has one item and one slice of K; the slices of an item
// are a cluster, whose sums meet in shared memory (in a fixed order), so a few rows of a long K still use many SMs and no
// partial sums go through memory.  The tiles of X and F travel by cp.async, ST stages deep.  With fewer than 64 rows the
// warps that have no rows take a share of K instead.
template <int RM, bool RCONTIG>
struct ShrinkTile {
    static constexpr int ST = RM >= 8 ? 3 : 4;
    static constexpr int XROW = 64 * 2 + 16;                                     // 64 of K; 16 bytes of padding: ldmatrix rows on different banks
    static constexpr int FROW = RCONTIG ? RM * 32 + 16 : XROW;
    static constexpr int XBYTES = kRows * XROW, FBYTES = (RCONTIG ? 64 : RM * 16) * FROW;
    static constexpr int PIPE = ST * (XBYTES + FBYTES), SUMS = kRows * RM * 16 * 4;
    static constexpr int BYTES = PIPE > SUMS ? PIPE : SUMS;
};
template <typename T, int RM, bool RCONTIG>
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const LoraParams p) {
    using S = ShrinkTile<RM, RCONTIG>;
    constexpr int PARTS = Split<T>::PARTS;
    extern __shared__ __align__(128) unsigned char smem[];
    chain_next();
    const Item it = find_item<kThreads>(p, blockIdx.x, p.rows_per_item);
    if (it.rows == 0 || it.adapter < 0) return;  // every CTA of the cluster
    const int splits = gridDim.y, split = blockIdx.y;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t sx = smem_u32(smem), sf = sx + S::ST * S::XBYTES;
    const T* x = static_cast<const T*>(p.x) + (long long)it.first * p.stride_x;
    const T* f = static_cast<const T*>(p.factor) + (long long)it.adapter * p.R * p.K;
    const int mt = (it.rows + 15) / 16;
    const int wm = mt > 2 ? 4 : mt, wk = 4 / wm;  // warps along the rows, along K
    const int m = warp % wm, phase = warp / wm;
    const int steps = (p.K + 63) / 64, per = (steps + splits - 1) / splits;
    const int step0 = min(split * per, steps), n = min(per, steps - step0);

    auto load = [&](int s) {
        if (s < n) {
            const int k0 = (step0 + s) * 64, st = s % S::ST;
            for (int c = t; c < mt * 16 * 8; c += kThreads) {
                const int row = c >> 3, k = k0 + (c & 7) * 8;
                const bool real = row < it.rows && k < p.K;
                cp16(sx + st * S::XBYTES + row * S::XROW + (c & 7) * 16, real ? x + row * p.stride_x + k : x, real);
            }
            if constexpr (RCONTIG) {
                for (int c = t; c < 64 * RM * 2; c += kThreads) {
                    const int k = c / (RM * 2), r = (c % (RM * 2)) * 8;
                    const bool real = k0 + k < p.K && r < p.R;
                    cp16(sf + st * S::FBYTES + k * S::FROW + r * 2, real ? f + (long long)(k0 + k) * p.R + r : f, real);
                }
            } else {
                for (int c = t; c < RM * 16 * 8; c += kThreads) {
                    const int r = c >> 3, k = k0 + (c & 7) * 8;
                    const bool real = k < p.K && r < p.R;
                    cp16(sf + st * S::FBYTES + r * S::FROW + (c & 7) * 16, real ? f + (long long)r * p.K + k : f, real);
                }
            }
        }
        cp_commit();
    };

    float acc[RM * 2][4];
#pragma unroll
    for (int i = 0; i < RM * 2; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
    for (int s = 0; s < S::ST - 1; ++s) load(s);
    for (int s = 0; s < n; ++s) {
        cp_wait<S::ST - 2>();
        __syncthreads();
        load(s + S::ST - 1);
        const uint32_t xs = sx + (s % S::ST) * S::XBYTES, fs = sf + (s % S::ST) * S::FBYTES;
        if (m < mt)
            for (int kk = phase; kk < 4; kk += wk) {
                uint32_t a[4];
                ldsm4(a, xs + (m * 16 + (lane & 15)) * S::XROW + kk * 32 + (lane >> 4) * 16);
#pragma unroll
                for (int r = 0; r < RM; ++r) {
                    uint32_t b[4];
                    if constexpr (RCONTIG)
                        ldsm4t(b, fs + (kk * 16 + (lane & 15)) * S::FROW + r * 32 + (lane >> 4) * 16);
                    else
                        ldsm4(b, fs + (r * 16 + (lane & 7) + (lane >> 4) * 8) * S::FROW + kk * 32 + ((lane >> 3) & 1) * 16);
                    mma16816<T>(acc[2 * r], a, b[0], b[1]);
                    mma16816<T>(acc[2 * r + 1], a, b[2], b[3]);
                }
            }
    }
    cp_wait<0>();
    __syncthreads();

    // the warps' shares of K, then the cluster's
    float* sums = reinterpret_cast<float*>(smem);  // [rows][RM * 16]
    constexpr int LD = RM * 16;
    for (int q = 0; q < wk; ++q) {
        if (q == phase && m < mt) {
#pragma unroll
            for (int i = 0; i < RM * 2; ++i) {
                float* at = sums + (m * 16 + (lane >> 2)) * LD + i * 8 + (lane & 3) * 2;
                float2* up = reinterpret_cast<float2*>(at);
                float2* dn = reinterpret_cast<float2*>(at + 8 * LD);
                float2 u = make_float2(acc[i][0], acc[i][1]), d = make_float2(acc[i][2], acc[i][3]);
                if (q) {
                    u.x += up->x; u.y += up->y;
                    d.x += dn->x; d.y += dn->y;
                }
                *up = u;
                *dn = d;
            }
        }
        __syncthreads();
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync();
    const float scale = p.scale ? __ldg(p.scale + it.adapter) : 1.f;
    // LANES neighbours have a row, each a pair of its ranks (two at RM 8)
    constexpr int LANES = RM == 1 ? 8 : RM == 2 ? 16 : 32, EACH = RM * 8 / LANES, TEAMS = kThreads / LANES;
    for (int r0 = split * TEAMS; r0 < it.rows; r0 += splits * TEAMS) {
        const int row = r0 + t / LANES;
        float2 v[EACH];
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = (t % LANES + i * LANES) * 2;
            v[i] = make_float2(0.f, 0.f);
            if (row < it.rows && r < p.R)
                for (int q = 0; q < splits; ++q) {
                    const float* from = splits > 1 ? cluster.map_shared_rank(sums, q) : sums;
                    const float2 u = *reinterpret_cast<const float2*>(from + row * LD + r);
                    v[i].x += u.x; v[i].y += u.y;
                }
            v[i].x *= scale; v[i].y *= scale;
            big = fmaxf(big, fmaxf(finite_abs(v[i].x), finite_abs(v[i].y)));
        }
        float down = 1.f;
        if constexpr (Split<T>::SCALED) {
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const int e = row_exponent(big);
            down = exp2_of(-e);
            if (t % LANES == 0 && row < it.rows) p.row_scale[it.first + row] = exp2_of(e);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = (t % LANES + i * LANES) * 2;
            if (row >= it.rows || r >= p.R) continue;
            uint32_t part[PARTS];
            split_pair<T>(v[i].x * down, v[i].y * down, part);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) *reinterpret_cast<uint32_t*>(static_cast<char*>(p.v) + k * plane_bytes(p.T, p.R) + ((long long)(it.first + row) * p.R + r) * 2) = part[k];
        }
    }
    if (splits > 1) cluster.sync();  // nobody's shared memory goes while others read it
}

// ------------------------------------------------------------------------------------------------------------------ expand
// out[t, c] = base[t, c] + sum_r v[t, r] G_a[c, r].  A CTA keeps its item's v as matrix operands in registers
// and walks over its columns, BN at a time, two tiles of G in shared memory.  The columns of a matrix instruction are
// permuted (its operand rows may come from anywhere) so that a thread's results are eight neighbours: base and out are then
// read and written 16 bytes at a time straight from and to memory.  Warps without rows take a share of the columns.
template <int RM, bool CCONTIG>
struct ExpandTile {
    static constexpr int BN = RM >= 8 ? 64 : 128;
    static constexpr int GROW = CCONTIG ? BN * 2 + 16 : RM * 32 + 16;
    // [c][r] rows: 32 bytes more every eight rows, because a matrix operand's rows are 0, 1, 8, 9, 16, 17, 24, 25
    static constexpr int GBYTES = CCONTIG ? RM * 16 * GROW : BN * GROW + BN / 8 * 32;
    static constexpr int BYTES = 2 * GBYTES;
    static constexpr int CHUNKS = RM * 16 * BN / 8 / kThreads;  // 16-byte pieces per thread and tile
};
template <typename T, int RM, bool CCONTIG>
__global__ void __launch_bounds__(kThreads) lora_expand_kernel(const LoraParams p) {
    using S = ExpandTile<RM, CCONTIG>;
    constexpr int BN = S::BN, PARTS = Split<T>::PARTS;
    extern __shared__ __align__(128) unsigned char smem[];
    const Item it = find_item<kThreads>(p, blockIdx.y, p.rows_per_item);
    if (it.rows == 0) return;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int col0 = blockIdx.x * p.cols_per_cta, col1 = min(col0 + p.cols_per_cta, p.K);
    const T* base = static_cast<const T*>(p.x);
    T* out = static_cast<T*>(p.out);
    if (it.adapter < 0) {  // base alone (zeros without one)
        chain_wait();
        if (base == out) return;
        const int n = (col1 - col0) / 8;
        for (int e = t; e < it.rows * n; e += kThreads) {
            const int row = e / n, c = col0 + (e - row * n) * 8;
            const uint4 v = base ? *reinterpret_cast<const uint4*>(base + (it.first + row) * p.stride_x + c) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + (it.first + row) * p.stride_out + c) = v;
        }
        return;
    }
    const T* g = static_cast<const T*>(p.factor) + (long long)it.adapter * p.R * p.K;
    const uint32_t sg = smem_u32(smem);
    const int mt = (it.rows + 15) / 16;
    const int wm = mt > 2 ? 4 : mt, wn = 4 / wm;
    const int m = warp % wm, share = warp / wm;
    const int tiles = (col1 - col0 + BN - 1) / BN;

    uint4 held[CCONTIG ? S::CHUNKS : 1];
    auto issue = [&](int tile) {  // [c][r]: straight to shared memory; [r][c]: to registers
        if (tile < tiles) {
            const int c0 = col0 + tile * BN;
#pragma unroll
            for (int i = 0; i < S::CHUNKS; ++i) {
                const int e = i * kThreads + t;
                if constexpr (CCONTIG) {
                    const int r = e / (BN / 8), c = c0 + e % (BN / 8) * 8;
                    held[i] = r < p.R && c < col1 ? __ldg(reinterpret_cast<const uint4*>(g + (long long)r * p.K + c)) : make_uint4(0, 0, 0, 0);
                } else {
                    const int c = e / (RM * 2), r = e % (RM * 2) * 8;
                    const bool real = r < p.R && c0 + c < col1;
                    cp16(sg + (tile & 1) * S::GBYTES + c * S::GROW + (c >> 3) * 32 + r * 2, real ? g + (long long)(c0 + c) * p.R + r : g, real);
                }
            }
        }
        if constexpr (!CCONTIG) cp_commit();
    };
    auto land = [&](int tile) {
        if constexpr (CCONTIG) {
            // column pair j of the 16-byte piece q of a group of 32 goes to word 4 j + q: the permutation of the columns
#pragma unroll
            for (int i = 0; i < S::CHUNKS; ++i) {
                const int e = i * kThreads + t, r = e / (BN / 8), q = e % (BN / 8);
                uint32_t* w = reinterpret_cast<uint32_t*>(smem + (tile & 1) * S::GBYTES + r * S::GROW) + q / 4 * 16 + q % 4;
                w[0] = held[i].x; w[4] = held[i].y; w[8] = held[i].z; w[12] = held[i].w;
            }
        } else {
            cp_wait<0>();
        }
    };
    issue(0);

    const int row0 = m * 16 + (lane >> 2), row1 = row0 + 8;
    const long long at0 = (long long)(it.first + row0), at1 = (long long)(it.first + row1);
    // base of the warp's groups of 32 columns of a tile, fetched a tile ahead
    constexpr int GROUPS = BN / 32;
    uint4 b0[GROUPS], b1[GROUPS];
    auto fetch = [&](int tile) {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int q = share + i * wn, c = col0 + tile * BN + q * 32 + (lane & 3) * 8;
            const bool on = base && tile < tiles && q < GROUPS && c < col1;
            b0[i] = on && row0 < it.rows ? *reinterpret_cast<const uint4*>(base + at0 * p.stride_x + c) : make_uint4(0, 0, 0, 0);
            b1[i] = on && row1 < it.rows ? *reinterpret_cast<const uint4*>(base + at1 * p.stride_x + c) : make_uint4(0, 0, 0, 0);
        }
    };
    fetch(0);
    chain_wait();
    uint32_t v[PARTS][RM][4];
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        const char* plane = static_cast<const char*>(p.v) + part * plane_bytes(p.T, p.R);
#pragma unroll
        for (int k = 0; k < RM; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i & 1 ? row1 : row0, r = k * 16 + (i >> 1) * 8 + (lane & 3) * 2;
                const bool real = row < it.rows && r < p.R;
                v[part][k][i] = real ? *reinterpret_cast<const uint32_t*>(plane + ((long long)(it.first + row) * p.R + r) * 2) : 0u;
            }
    }
    float f0 = 1.f, f1 = 1.f;  // the rows' powers of two
    if constexpr (Split<T>::SCALED) {
        if (row0 < it.rows) f0 = p.row_scale[at0];
        if (row1 < it.rows) f1 = p.row_scale[at1];
    }
    for (int tile = 0; tile < tiles; ++tile) {
        const int c0 = col0 + tile * BN;
        land(tile);
        __syncthreads();
        issue(tile + 1);
        const unsigned char* gs = smem + (tile & 1) * S::GBYTES;
#pragma unroll
        for (int g32 = 0; g32 < GROUPS; ++g32) {
            const int q = share + g32 * wn;
            if (m >= mt || q >= GROUPS) break;
            const int c = c0 + q * 32 + (lane & 3) * 8;
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
            for (int k = 0; k < RM; ++k) {
                uint32_t b[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // instructions 2h and 2h + 1 of the four
                    if constexpr (CCONTIG) {
                        ldsm4t(b[h], smem_u32(gs) + (k * 16 + (lane & 15)) * S::GROW + q * 64 + h * 32 + (lane >> 4) * 16);
                    } else {
                        const int j = 2 * h + (lane >> 4), i = lane & 7;
                        const int n = q * 32 + (i >> 1) * 8 + j * 2 + (i & 1);
                        ldsm4(b[h], smem_u32(gs) + n * S::GROW + (n >> 3) * 32 + k * 32 + ((lane >> 3) & 1) * 16);
                    }
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma16816<T>(acc[2 * h], v[part][k], b[h][0], b[h][1]);
                        mma16816<T>(acc[2 * h + 1], v[part][k], b[h][2], b[h][3]);
                    }
            }
            auto joined = [&](const uint4& b, int o) {
                const uint32_t in[4] = {b.x, b.y, b.z, b.w};
                const float f = o ? f1 : f0;
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 u = unpack2<T>(in[j]);
                    r[j] = pack2<T>(fmaf(acc[j][o], f, u.x), fmaf(acc[j][o + 1], f, u.y));
                }
                return make_uint4(r[0], r[1], r[2], r[3]);
            };
            if (row0 < it.rows && c < col1) *reinterpret_cast<uint4*>(out + at0 * p.stride_out + c) = joined(b0[g32], 0);
            if (row1 < it.rows && c < col1) *reinterpret_cast<uint4*>(out + at1 * p.stride_out + c) = joined(b1[g32], 2);
        }
        fetch(tile + 1);
    }
}

// ---------------------------------------------------------------------------------------------------------------- few rows
// Both products of the forward pass in one kernel, for items of at most 16 rows.  A cluster of eight CTAs has an item: each
// CTA takes an eighth of the contraction of h, the eight sums meet through shared memory, and each CTA multiplies the whole
// h with its own columns' part of U, which has been on its way into shared memory since the kernel began.  Both products run
// on m16n8k16 with the order of k chosen so that a thread's operands are 16 (8) consecutive bytes: any order will do as long
// as both operands have the same.  The columns of four neighbouring tiles are dealt out so that a thread ends with eight
// consecutive ones.
// Bound: latency (index, operands, two cluster barriers, store); what is read again is read from L2.
struct FewParams {
    LoraParams l;  // x, K: of h; factor: D; out
    const void* base; const void* up;
    long long stride_base;
    int N, cols;  // columns of a CTA, a multiple of 32
};
constexpr int kFewRows = 16, kFewWarps = 8, kFewCluster = 8;
// CTAs per SM that the registers leave room for
constexpr int few_per_sm(int R) { return R <= 64 ? 2 : 1; }
template <int R>
struct FewTile {
    static constexpr int LDH = R + 8;
    // groups of warps that share the ranks in the first product (a warp has its sums and its steps of D in registers), tiles of
    // eight ranks of a group, groups along k
    static constexpr int GROUPS = R <= 32 ? 1 : R <= 64 ? 2 : 4, NT = (R / 8 + GROUPS - 1) / GROUPS, KW = kFewWarps / GROUPS;
    static constexpr int RED = KW * 16 * R * 4, PART = 16 * R * 4;
    template <typename T>
    static constexpr int H = Split<T>::PARTS * 16 * LDH * 2 + 16 * 4;  // the parts of h, the rows' powers of two
    template <typename T>
    static int bytes(int cols) { return cols * R * 2 + RED + PART + H<T>; }
    // 16-byte piece of U's row: pieces that half a warp reads together are on different banks
    static __device__ __forceinline__ int piece(int row, int ch) {
        const int far = (row >> 3) & 1;
        if (R == 16) return (row ^ (far << 1)) * 2 + ch;
        if (R == 32) return row * 4 + (ch ^ (far << 1));
        if (R == 64) return row * 8 + (ch ^ ((row & 1) << 1) ^ (far << 2));
        return row * (R / 8) + ch;
    }
};
template <typename T, int R>
__global__ void __launch_bounds__(kFewWarps * 32, few_per_sm(R)) lora_few_kernel(const FewParams f) {
    using S = FewTile<R>;
    constexpr int PARTS = Split<T>::PARTS;
    extern __shared__ __align__(16) unsigned char few_smem[];
    const LoraParams& p = f.l;
    const Item it = find_item<kFewWarps * 32>(p, blockIdx.x, kFewRows);
    if (it.rows == 0) return;  // every CTA of the cluster
    const int col0 = blockIdx.y * f.cols, ncols = max(0, min(f.cols, f.N - col0));
    const T* base = f.base ? static_cast<const T*>(f.base) + it.first * f.stride_base + col0 : nullptr;
    T* out = static_cast<T*>(p.out) + it.first * p.stride_out + col0;
    if (it.adapter < 0) {  // base alone (zeros without one)
        if (base == out) return;
        for (int e = threadIdx.x; e < it.rows * (ncols / 8); e += kFewWarps * 32) {
            const int row = e / (ncols / 8), c = (e - row * (ncols / 8)) * 8;
            const uint4 v = base ? *reinterpret_cast<const uint4*>(base + row * f.stride_base + c) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + row * p.stride_out + c) = v;
        }
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* us = few_smem;
    float* red = reinterpret_cast<float*>(few_smem + (size_t)f.cols * R * 2);
    float* part = red + S::RED / 4;
    float* powers = part + S::PART / 4;
    T* hs = reinterpret_cast<T*>(powers + 16);
    const bool on0 = g < it.rows, on1 = g + 8 < it.rows;
    // this CTA's part of h: 32 values of k per step
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    const int slice = (p.K + 32 * kFewCluster - 1) / (32 * kFewCluster) * 32, k1 = min((rank + 1) * slice, p.K);
    const T* x0 = static_cast<const T*>(p.x) + (it.first + g) * p.stride_x;
    const T* x1 = x0 + 8 * p.stride_x;
    const int kw = warp % S::KW, r0 = warp / S::KW * (S::NT * 8);
    const T* d0 = static_cast<const T*>(p.factor) + ((long long)it.adapter * R + r0 + g) * p.K;
    constexpr int DEPTH = R == 16 ? 3 : 2, STEP = S::KW * 32, NT = S::NT;  // steps on their way
    uint4 xa[DEPTH], xb[DEPTH], d[DEPTH][NT];
    auto load = [&](int i, int k0) {
        const int k = k0 + t * 8;
        const bool in = k < k1;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        xa[i] = in && on0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
        xb[i] = in && on1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) d[i][n] = in && r0 + n * 8 < R ? __ldg(reinterpret_cast<const uint4*>(d0 + (long long)n * 8 * p.K + k)) : zero;
    };
    const int first = rank * slice + kw * 32;
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) load(i, first + i * STEP);
    // U and base under their latency
    {
        const T* u = static_cast<const T*>(f.up) + ((long long)it.adapter * f.N + col0) * R;
        const uint32_t to = smem_u32(us);
        for (int e = threadIdx.x; e < ncols * (R / 8); e += kFewWarps * 32) {
            const int row = e / (R / 8), ch = e % (R / 8);
            cp16(to + S::piece(row, ch) * 16, u + (long long)e * 8, true);
        }
        cp_commit();
    }
    // the first blocks of base: a warp has every eighth block of 32 columns
    constexpr int AHEAD = 3;
    const int blocks = (ncols + 31) / 32;
    uint4 b0[AHEAD], b1[AHEAD];
    auto fetch = [&](int i, int blk) {
        const int c = blk * 32 + t * 8;
        const bool in = base && c < ncols;
        b0[i] = in && on0 ? *reinterpret_cast<const uint4*>(base + g * f.stride_base + c) : make_uint4(0, 0, 0, 0);
        b1[i] = in && on1 ? *reinterpret_cast<const uint4*>(base + (g + 8) * f.stride_base + c) : make_uint4(0, 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(i, warp + i * kFewWarps);

    float acc[NT][4] = {};
    for (int k0 = first; k0 < k1; k0 += DEPTH * STEP) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (k0 + i * STEP >= k1) break;
            const uint32_t a0[4] = {xa[i].x, xb[i].x, xa[i].y, xb[i].y}, a1[4] = {xa[i].z, xb[i].z, xa[i].w, xb[i].w};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma16816<T>(acc[n], a0, d[i][n].x, d[i][n].y);
                mma16816<T>(acc[n], a1, d[i][n].z, d[i][n].w);
            }
            load(i, k0 + (i + DEPTH) * STEP);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (r0 + n * 8 >= R) break;  // (the last group may have fewer)
        float* at = red + (kw * 16 + g) * R + r0 + n * 8 + t * 2;
        *reinterpret_cast<float2*>(at) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(at + 8 * R) = make_float2(acc[n][2], acc[n][3]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * R; e += kFewWarps * 32) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < S::KW; ++w) s += red[w * 16 * R + e];
        part[e] = s;
    }
    const float scale = p.scale ? __ldg(p.scale + it.adapter) : 1.f;
    cluster.sync();
    // LANES neighbours have a row
    constexpr int LANES = R == 16 ? 16 : 32, EACH = (R + LANES - 1) / LANES, TEAMS = kFewWarps * 32 / LANES;
#pragma unroll
    for (int r0 = 0; r0 < kFewRows; r0 += TEAMS) {
        const int row = r0 + threadIdx.x / LANES, l = threadIdx.x % LANES;
        float h[EACH], big = 0.f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = l + i * LANES;
            float v[kFewCluster];
            h[i] = 0.f;
            if (R % LANES && r >= R) continue;
#pragma unroll
            for (int q = 0; q < kFewCluster; ++q) v[q] = cluster.map_shared_rank(part, q)[row * R + r];
#pragma unroll
            for (int q = 0; q < kFewCluster; ++q) h[i] += v[q];
            h[i] *= scale;
            big = fmaxf(big, finite_abs(h[i]));
        }
        float down = 1.f;
        if constexpr (Split<T>::SCALED) {
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const int e = row_exponent(big);
            down = exp2_of(-e);
            if (l == 0) powers[row] = exp2_of(e);
            if (l == 0 && blockIdx.y == 0 && row < it.rows) p.row_scale[it.first + row] = exp2_of(e);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = l + i * LANES;
            if (R % LANES && r >= R) continue;
            uint32_t words[PARTS];
            split_pair<T>(h[i] * down, 0.f, words);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
                const T one = from_f32<T>(unpack2<T>(words[k]).x);
                hs[(k * 16 + row) * S::LDH + r] = one;
                if (blockIdx.y == 0 && row < it.rows)  // for the backward pass
                    reinterpret_cast<T*>(static_cast<char*>(p.v) + k * plane_bytes(p.T, p.R))[(long long)(it.first + row) * R + r] = one;
            }
        }
    }
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // the others' sums have been read
    cp_wait<0>();
    __syncthreads();

    uint32_t a[PARTS][R / 16][4];
#pragma unroll
    for (int v = 0; v < PARTS; ++v)
#pragma unroll
        for (int s = 0; s < R / 16; ++s) {
            const uint2 lo8 = *reinterpret_cast<const uint2*>(hs + (v * 16 + g) * S::LDH + s * 16 + t * 4);
            const uint2 hi8 = *reinterpret_cast<const uint2*>(hs + (v * 16 + g + 8) * S::LDH + s * 16 + t * 4);
            a[v][s][0] = lo8.x; a[v][s][1] = hi8.x; a[v][s][2] = lo8.y; a[v][s][3] = hi8.y;
        }
    const float f0 = Split<T>::SCALED ? powers[g] : 1.f, f1 = Split<T>::SCALED ? powers[g + 8] : 1.f;
    for (int blk0 = warp; blk0 < blocks; blk0 += AHEAD * kFewWarps) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int blk = blk0 + i * kFewWarps;
            if (blk >= blocks) break;
            float o[4][4] = {};
#pragma unroll
            for (int s = 0; s < R / 16; ++s) {
                uint2 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // column n of tile j; behind the last column: some other row of U, whose result is not stored
                    const int row = min(blk * 32 + (g >> 1) * 8 + j * 2 + (g & 1), ncols - 1);
                    b[j] = *reinterpret_cast<const uint2*>(us + S::piece(row, s * 2 + (t >> 1)) * 16 + (t & 1) * 8);
                }
#pragma unroll
                for (int v = 0; v < PARTS; ++v)  // (neighbouring instructions do not wait for one another)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma16816<T>(o[j], a[v][s], b[j].x, b[j].y);
            }
            auto joined = [&](const uint4& b, int at) {
                const uint32_t in[4] = {b.x, b.y, b.z, b.w};
                const float f = at ? f1 : f0;
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = unpack2<T>(in[j]);
                    r[j] = pack2<T>(fmaf(o[j][at], f, v.x), fmaf(o[j][at + 1], f, v.y));
                }
                return make_uint4(r[0], r[1], r[2], r[3]);
            };
            const int c = blk * 32 + t * 8;
            if (c < ncols && on0) *reinterpret_cast<uint4*>(out + g * p.stride_out + c) = joined(b0[i], 0);
            if (c < ncols && on1) *reinterpret_cast<uint4*>(out + (g + 8) * p.stride_out + c) = joined(b1[i], 2);
            fetch(i, blk + AHEAD * kFewWarps);
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------------------------- outer
// part[item][r, k] = sum over the item's rows of v[t, r] X[t, k] ([k, r] with KROWS, job 0), fp32, for one item of up to
// rows_per_item rows and 128 columns.  Both operands are transposed on the way from shared memory to registers.
template <typename T, int RM>
struct OuterTile {
    static constexpr int PARTS = Split<T>::PARTS, ST = PARTS * RM >= 12 ? 3 : 4, BT = 32;
    static constexpr int XROW = 128 * 2 + 16, VROW = RM * 32 + 16;
    static constexpr int XBYTES = BT * XROW, VBYTES = BT * VROW;
    static constexpr int POWERS = XBYTES + PARTS * VBYTES;  // the rows' powers of two
    static constexpr int STAGE = POWERS + (Split<T>::SCALED ? BT * 4 : 0), BYTES = ST * STAGE;
};
template <typename T, int RM, bool KROWS>
__device__ __forceinline__ void outer_product(const LoraParams& p, const OuterJob& job, const Item& it, int w, int c0, unsigned char* smem) {
    using S = OuterTile<T, RM>;
    constexpr int PARTS = S::PARTS;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const T* x = static_cast<const T*>(job.x) + (long long)it.first * job.stride_x;
    const char* v0 = static_cast<const char*>(job.v) + (long long)it.first * p.R * 2;
    const uint32_t sm = smem_u32(smem);
    const int n = (it.rows + S::BT - 1) / S::BT;

    auto load = [&](int s) {
        if (s < n) {
            const int r0 = s * S::BT;
            const uint32_t st = sm + (s % S::ST) * S::STAGE;
#pragma unroll
            for (int i = 0; i < S::BT * 16 / kThreads; ++i) {
                const int e = i * kThreads + t, row = e >> 4, c = c0 + (e & 15) * 8;
                const bool real = r0 + row < it.rows && c < job.K;
                cp16(st + row * S::XROW + (e & 15) * 16, real ? x + (r0 + row) * job.stride_x + c : x, real);
            }
            for (int e = t; e < S::BT * RM * 2; e += kThreads) {
                const int row = e / (RM * 2), r = e % (RM * 2) * 8;
                const bool real = r0 + row < it.rows && r < p.R;
                const long long at = real ? ((long long)(r0 + row) * p.R + r) * 2 : 0;
#pragma unroll
                for (int k = 0; k < PARTS; ++k) cp16(st + S::XBYTES + k * S::VBYTES + row * S::VROW + r * 2, v0 + k * plane_bytes(p.T, p.R) + at, real);
            }
            if constexpr (Split<T>::SCALED)
                if (t < S::BT) cp4(st + S::POWERS + t * 4, job.row_scale + it.first + (r0 + t < it.rows ? r0 + t : 0));
        }
        cp_commit();
    };

    // !KROWS: rows of the accumulator are r (RM tiles of 16), columns the warp's 32 of X (4 tiles of 8)
    //  KROWS: rows are the warp's 32 columns of X (2 tiles of 16), columns are r (2 RM tiles of 8)
    constexpr int MI = KROWS ? 2 : RM, NI = KROWS ? 2 * RM : 4;
    float acc[MI][NI][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
#pragma unroll
    for (int s = 0; s < S::ST - 1; ++s) load(s);
    // the item's largest power of two, which its rows are brought to
    int top = 0;
    if constexpr (Split<T>::SCALED) {
        __shared__ int tops[kThreads / 32];
        top = -126;
        for (int r = t; r < it.rows; r += kThreads) top = max(top, (int)(__float_as_uint(job.row_scale[it.first + r]) >> 23) - 127);
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
        for (int w2 = 0; w2 < kThreads / 32; ++w2) top = max(top, tops[w2]);
    }
    for (int s = 0; s < n; ++s) {
        cp_wait<S::ST - 2>();
        __syncthreads();
        load(s + S::ST - 1);
        const uint32_t xs = sm + (s % S::ST) * S::STAGE + warp * 64, vs = sm + (s % S::ST) * S::STAGE + S::XBYTES;
#pragma unroll
        for (int tt = 0; tt < S::BT; tt += 16) {
            // operand with rows = columns of shared memory: matrices (t 0-7, c 0-7), (t 0-7, c 8-15), (t 8-15, ...) transposed
            const int arow = tt + (lane & 7) + (lane >> 4) * 8, acol = ((lane >> 3) & 1) * 16;
            const int brow = tt + (lane & 15), bcol = (lane >> 4) * 16;
            // ratios of this lane's rows tt + 2 (lane % 4) + {0, 1} and eight rows on to the item's power, in two factors each
            __half2 ratio[2][2];
            if constexpr (Split<T>::SCALED) {
                const float* f = reinterpret_cast<const float*>(smem + (s % S::ST) * S::STAGE + S::POWERS) + tt + (lane & 3) * 2;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float2 a, b;
                    row_ratio(f[i * 8], top, a.x, b.x);
                    row_ratio(f[i * 8 + 1], top, a.y, b.y);
                    ratio[i][0] = __float22half2_rn(a);
                    ratio[i][1] = __float22half2_rn(b);
                }
            }
            auto level = [&](uint32_t& w, int i) {
                if constexpr (Split<T>::SCALED) {
                    __half2 h = *reinterpret_cast<__half2*>(&w);
                    h = __hmul2(__hmul2(h, ratio[i][0]), ratio[i][1]);
                    w = *reinterpret_cast<uint32_t*>(&h);
                }
            };
            if constexpr (KROWS) {
                uint32_t a[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) ldsm4t(a[i], xs + arow * S::XROW + i * 32 + acol);
#pragma unroll
                for (int r = 0; r < RM; ++r)
#pragma unroll
                    for (int h = 0; h < PARTS; ++h) {
                        uint32_t b[4];
                        ldsm4t(b, vs + h * S::VBYTES + brow * S::VROW + r * 32 + bcol);
                        level(b[0], 0); level(b[1], 1); level(b[2], 0); level(b[3], 1);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            mma16816<T>(acc[i][2 * r], a[i], b[0], b[1]);
                            mma16816<T>(acc[i][2 * r + 1], a[i], b[2], b[3]);
                        }
                    }
            } else {
                uint32_t b[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) ldsm4t(b[j], xs + brow * S::XROW + j * 32 + bcol);
#pragma unroll
                for (int r = 0; r < RM; ++r)
#pragma unroll
                    for (int h = 0; h < PARTS; ++h) {
                        uint32_t a[4];
                        ldsm4t(a, vs + h * S::VBYTES + arow * S::VROW + r * 32 + acol);
                        level(a[0], 0); level(a[1], 0); level(a[2], 1); level(a[3], 1);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            mma16816<T>(acc[r][2 * j], a, b[j][0], b[j][1]);
                            mma16816<T>(acc[r][2 * j + 1], a, b[j][2], b[j][3]);
                        }
                    }
            }
        }
    }
    cp_wait<0>();
    float* part = job.part + (long long)w * p.R * job.K;
    const float up = Split<T>::SCALED ? exp2_of(top) : 1.f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const int mrow = i * 16 + (lane >> 2) + o * 8, ncol = j * 8 + (lane & 3) * 2;
                const float2 v = make_float2(acc[i][j][2 * o] * up, acc[i][j][2 * o + 1] * up);
                if constexpr (KROWS) {
                    const int k = c0 + warp * 32 + mrow;
                    if (k < job.K && ncol < p.R) *reinterpret_cast<float2*>(part + (long long)k * p.R + ncol) = v;
                } else {
                    const int k = c0 + warp * 32 + ncol;
                    if (k < job.K && mrow < p.R) *reinterpret_cast<float2*>(part + (long long)mrow * job.K + k) = v;
                }
            }
}

template <typename T, int RM>
__global__ void __launch_bounds__(kThreads) lora_outer_kernel(const LoraParams p, const __grid_constant__ OuterJobs jobs) {
    extern __shared__ __align__(128) unsigned char smem[];
    // last items first: their rows are the ones that the kernel before this one read last and left in the L2 cache
    const int group = (int)blockIdx.x - jobs.groups, which = group < 0 ? 0 : 1;
    const int w = jobs.job[which].items - 1 - (int)blockIdx.y;
    chain_next();
    const Item it = find_item<kThreads>(p, w, jobs.job[which].rows);
    chain_wait();
    if (w < 0) return;  // (the other job has more items)
    if ((blockIdx.x == 0 || group == 0) && threadIdx.x == 0) jobs.job[which].item_adapter[w] = it.rows ? it.adapter : -1;
    if (it.rows == 0 || it.adapter < 0) return;
    if (group < 0) outer_product<T, RM, true>(p, jobs.job[0], it, w, (int)blockIdx.x * 128, smem);
    else outer_product<T, RM, false>(p, jobs.job[1], it, w, group * 128, smem);
}

// dF[a] = sum of the partial products of a's items, in the items' order; zero for an adapter without rows.  One launch for
// both factors: `blocks` CTAs (of 1024 values each) for the first, the rest for the second.
template <typename T>
struct Join {
    const float* part;
    const int* item_adapter;
    T* out;
    long long size;
    int items, blocks;
};
template <typename T>
__global__ void __launch_bounds__(256) lora_join_kernel(const Join<T> first, const Join<T> second) {
    __shared__ int mine[256];
    __shared__ int count;
    chain_next();
    chain_wait();
    const bool one = (int)blockIdx.x < first.blocks;
    const Join<T>& j = one ? first : second;
    const int a = blockIdx.y, t = threadIdx.x;
    const long long at = ((long long)(one ? blockIdx.x : blockIdx.x - first.blocks) * 256 + t) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w0 = 0; w0 < j.items; w0 += 256) {
        __syncthreads();
        if (t < 32) {  // the items of this adapter, in order
            int n = 0;
            for (int w = w0; w < min(w0 + 256, j.items); w += 32) {
                const bool hit = w + t < j.items && j.item_adapter[w + t] == a;
                const unsigned b = __ballot_sync(0xffffffffu, hit);
                if (hit) mine[n + __popc(b & ((1u << t) - 1))] = w + t;
                n += __popc(b);
            }
            if (t == 0) count = n;
        }
        __syncthreads();
        if (at < j.size) {
#pragma unroll 4
            for (int i = 0; i < count; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(j.part + (long long)mine[i] * j.size + at);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        }
    }
    if (at < j.size) *reinterpret_cast<uint2*>(j.out + (long long)a * j.size + at) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

// --------------------------------------------------------------------------------------------------------------- launchers
// Whether a call runs on the tcgen05 kernels.  Their tiles are 128 rows and a launch costs some 3 us more, so the requests
// have to be long on the whole, and there has to be work: the mma.sync kernels fall behind with the rank (shared memory
// feeds their instructions) and, having 64-row items in clusters of eight, with a long contraction over few rows.  Measured,
// mma.sync / tcgen05, forward, bf16, K = 2048, N = 6144: rank 16: 512 rows 8.6 / 13.3 us, 8192 rows 54.4 / 51.5; rank 64: 512
// rows 17.8 / 13.4, 1024 rows 23.7 / 17.3; 64 requests of 32 rows 46.4 / 48.2, of 64 rows 67.7 / 59.8.  K = 12288, N = 3072, rank
// 32: 1300 rows 28.3 / 21.2 us.  Rank 128, K = 2048, N = 6144: 2048 rows of 32 requests 56.7 / 44.1 us, 512 rows of 16 31.1 / 31.2.
bool use_tc(const nb_lora_args* a) {
    if (a->impl != NB_IMPL_AUTO) return a->impl == NB_IMPL_TCGEN05;
    const int contraction = a->dy ? a->N : a->K;
    if (a->R >= 32 && contraction >= 8192 && a->T >= 16ll * a->requests) return true;
    if (a->R > 64 && a->T >= 48ll * a->requests) return true;
    return a->T >= 96ll * a->requests && (double)a->T * a->R * a->R * ((double)a->K + a->N) >= 1e10;
}
// Whether the forward pass is the one kernel for few rows: where its clusters are resident together, or in two turns when
// one cluster per item is enough (it then reads D once and still saves a kernel).  Two kernels / one, measured in bf16: rank 16,
// K = 3072, N = 18432: 1 row 6.9 / 5.2 us, 24 rows of 24 requests 13.0 / 9.8, 64 of 64 (two turns) 27.3 / 20.0; rank 32, K =
// 12288, N = 3072: 128 rows 15.9 (tcgen05) / 9.1, 1024 rows of 64 requests (two turns) 50.6 (tcgen05) / 24.5; rank 64, 128 rows of 4
// requests 16.3 (tcgen05) / 13.8; K = 2048, N = 6144, 1024 rows of 64 requests: rank 16 16.5 / 17.0, rank 32 22.8 / 20.2.  Not
// taken, before h had its present parts: rank 64, K = 3072, N = 18432 (four clusters per item), 256 rows 19.1 / 22.6; rank 32, 24
// rows of 24 requests (two clusters per item) 16.1 / 16.9.
int few_need(const nb_lora_args* a) {  // clusters of an item that keep a CTA's part of U within 80 KB
    return ceil_div((long long)a->N * a->R * 2, kFewCluster * 80 * 1024);
}
// CTAs that are resident together.  With one CTA per SM (above rank 64), clusters of eight do not fill the SMs: 16 clusters of
// rank 128 took two turns (8 rows of 8 requests, 12288 -> 3072, before h had its present parts: 25.9 us for 24.4), 8 one (128 rows at rank 80:
// 17.0 for 17.5 on tcgen05).
int few_slots(int R) { return R <= 64 ? 2 * sms() : 3 * sms() / 4; }
bool use_few(const nb_lora_args* a) {
    if (a->impl == NB_IMPL_TCGEN05) return false;
    const long long tiles = ceil_div(a->T, kFewRows), requests = a->requests < a->T ? a->requests : a->T;
    const int need = few_need(a);
    return (tiles > requests ? tiles : requests) * need * kFewCluster <= (long long)few_slots(a->R) * (need == 1 && a->R <= 64 ? 2 : 1);
}
// A tcgen05 launch, or the mma.sync one where there is no tensor map for the operands (rows a stride of zero apart) and the
// caller did not insist.
#define NB_TC_OR(a, tc_call, call)                                                                             \
    ([&]() -> int {                                                                                            \
        if (!use_tc(a)) return call;                                                                           \
        const int rc_ = tc_call;                                                                               \
        return rc_ == NB_ERR_UNSUPPORTED && (a)->impl == NB_IMPL_AUTO ? call : rc_;                            \
    }())
// rows of the gradients' items: long enough that the partial products stay small beside the operands, short enough that the
// CTAs cover the SMs: one wave of one per SM (an item and 256 columns each) with the tcgen05 kernels, about four per SM (128
// columns) with the small ones
int outer_rows(const nb_lora_args* a, int cols) {
    int want = use_tc(a) ? sms() / ceil_div(cols, kTcCols) : ceil_div(4ll * sms(), ceil_div(cols, 128));
    if (want < 1) want = 1;
    const int rows = ceil_div(ceil_div(a->T, want), 64) * 64;
    return rows < 128 ? 128 : rows;
}

template <typename K>
int allow_smem(K kernel, int bytes) {
    if (bytes > 48 * 1024) NB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return NB_OK;
}

template <typename T, int RM, bool RCONTIG>
int shrink(const LoraParams& p, cudaStream_t s) {
    using S = ShrinkTile<RM, RCONTIG>;
    const int items = item_count(p.T, p.requests, kRows);
    // CTAs of an item: a power of two up to eight (a portable cluster), until the items cover the SMs twice, each with at
    // least two steps of 64 of K
    const int live = live_items(p, kRows);
    int splits = 1;
    while (splits < 8 && live * splits < 2 * sms() && ceil_div(p.K, 64) >= 4 * splits) splits *= 2;
    auto* kernel = lora_shrink_kernel<T, RM, RCONTIG>;
    if (int rc = allow_smem(kernel, S::BYTES)) return rc;
    return launch(kernel, dim3(items, splits), kThreads, S::BYTES, splits, p.chained, s, p);
}
template <typename T, int RM, bool CCONTIG>
int expand(LoraParams p, cudaStream_t s) {
    using S = ExpandTile<RM, CCONTIG>;
    const int items = item_count(p.T, p.requests, kRows);
    const int live = live_items(p, kRows);
    // columns of a CTA: whole tiles, as many as leave about four CTAs per SM: they are resident together (measured
    // with 24 rows of 24 requests, 3072 -> 18432, rank 16: 12.8 us for both products, 14.5 with eight per SM in two waves, 14.5
    // with two)
    const int tiles = ceil_div(p.K, S::BN), per = ceil_div(4ll * sms(), live);
    p.cols_per_cta = ceil_div(tiles, per < tiles ? per : tiles) * S::BN;
    auto* kernel = lora_expand_kernel<T, RM, CCONTIG>;
    if (int rc = allow_smem(kernel, S::BYTES)) return rc;
    return launch(kernel, dim3(ceil_div(p.K, p.cols_per_cta), items), kThreads, S::BYTES, 1, p.chained, s, p);
}
template <typename T, int R>
int few(const nb_lora_args* a, const LoraParams& p, cudaStream_t s) {
    FewParams f = {};
    f.l = p;
    f.l.x = a->x; f.l.stride_x = a->stride_x; f.l.factor = a->down; f.l.K = a->K;
    f.l.out = a->out; f.l.stride_out = a->stride_out;
    f.base = a->base; f.stride_base = a->stride_base; f.up = a->up; f.N = a->N;
    // clusters of an item: more than it needs where few items leave SMs idle, each of which computes h anew, as long as that
    // reads less than its columns
    const int live = live_items(f.l, kFewRows), need = few_need(a);
    int splits = few_slots(R) / (kFewCluster * live);
    if (splits > ceil_div(a->N, a->K)) splits = ceil_div(a->N, a->K);
    if (splits < need) splits = need;
    f.cols = ceil_div(ceil_div(a->N, kFewCluster * splits), 32) * 32;
    auto* kernel = lora_few_kernel<T, R>;
    const int bytes = FewTile<R>::template bytes<T>(f.cols);
    if (int rc = allow_smem(kernel, bytes)) return rc;
    return launch(kernel, dim3(item_count(a->T, a->requests, kFewRows), kFewCluster * splits), kFewWarps * 32, bytes, kFewCluster, false, s, f);
}
template <typename T, int RM>
int outer(const nb_lora_args* a, const LoraParams& p, OuterJobs j, cudaStream_t s) {
    using S = OuterTile<T, RM>;
    auto small = [&]() -> int {
        auto* kernel = lora_outer_kernel<T, RM>;
        if (int rc = allow_smem(kernel, S::BYTES)) return rc;
        j.groups = ceil_div(j.job[0].K, 128);
        const int groups = j.groups + ceil_div(j.job[1].K, 128);
        const int items = j.job[0].items > j.job[1].items ? j.job[0].items : j.job[1].items;
        return launch(kernel, dim3(groups, items), kThreads, S::BYTES, 1, p.chained, s, p, j);
    };
    return NB_TC_OR(a, tc_outer(p, j, a->dtype, s), small());
}

// The gradients' workspace: for each of the two factors asked for, the items' adapters and their partial products.
struct Piece {
    int64_t table, part, end;
    int rows, items;
};
Piece piece_of(const nb_lora_args* a, int cols, int64_t at) {
    Piece p;
    p.rows = outer_rows(a, cols);
    p.items = item_count(a->T, a->requests, p.rows);
    p.table = at;
    p.part = at + ((int64_t)p.items * 4 + 255) / 256 * 256;
    p.end = p.part + ((int64_t)p.items * a->R * cols * 4 + 255) / 256 * 256;
    return p;
}

LoraParams params_of(const nb_lora_args* a) {
    LoraParams p = {};
    p.offsets = a->offsets; p.adapters = a->adapters; p.scale = a->scale;
    p.T = a->T; p.R = a->R; p.A = a->A; p.requests = a->requests;
    p.rows_per_item = kRows;
    p.status = static_cast<int*>(a->status);
    return p;
}
float* powers_of(void* h, const nb_lora_args* a) { return reinterpret_cast<float*>(static_cast<char*>(h) + parts_of(a->dtype) * plane_bytes(a->T, a->R)); }

template <typename T, int RM>
int forward_t(const nb_lora_args* a, cudaStream_t s) {
    LoraParams p = params_of(a);
    p.v = a->h;
    p.row_scale = powers_of(a->h, a);
    if (use_few(a)) switch (a->R) {
            case 16: return few<T, 16>(a, p, s);
            case 32: return few<T, 32>(a, p, s);
            case 48: return few<T, 48>(a, p, s);
            case 64: return few<T, 64>(a, p, s);
            case 80: return few<T, 80>(a, p, s);
            case 96: return few<T, 96>(a, p, s);
            case 112: return few<T, 112>(a, p, s);
            default: return few<T, 128>(a, p, s);
        }
    p.x = a->x; p.stride_x = a->stride_x; p.factor = a->down; p.K = a->K;
    if (int rc = NB_TC_OR(a, tc_shrink(p, false, a->dtype, s), (shrink<T, RM, false>(p, s)))) return rc;
    p.chained = true;
    p.x = a->base; p.stride_x = a->stride_base; p.out = a->out; p.stride_out = a->stride_out; p.factor = a->up; p.K = a->N;
    return NB_TC_OR(a, tc_expand(p, false, a->dtype, s), (expand<T, RM, false>(p, s)));
}
template <typename T, int RM>
int backward_t(const nb_lora_args* a, cudaStream_t s) {
    LoraParams g = params_of(a);
    if (a->dx || a->ddown) {
        g.v = a->g;
        g.row_scale = powers_of(a->g, a);
        g.x = a->dy; g.stride_x = a->stride_dy; g.factor = a->up; g.K = a->N;
        if (int rc = NB_TC_OR(a, tc_shrink(g, true, a->dtype, s), (shrink<T, RM, true>(g, s)))) return rc;
    }
    g.chained = a->dx || a->ddown;
    if (a->dup || a->ddown) {
        char* ws = static_cast<char*>(a->workspace);
        int64_t used = 0;
        OuterJobs j = {};
        Join<T> joins[2] = {};
        int n = 0;
        auto job = [&](int i, const void* x, long long stride, int cols, void* planes, void* grad) {
            const Piece w = piece_of(a, cols, used);
            used = w.end;
            float* part = reinterpret_cast<float*>(ws + w.part);
            int* table = reinterpret_cast<int*>(ws + w.table);
            j.job[i] = {x, planes, powers_of(planes, a), part, table, stride, cols, w.rows, w.items};
            const long long size = (long long)a->R * cols;
            joins[n++] = {part, table, static_cast<T*>(grad), size, w.items, ceil_div(size, 1024)};
        };
        if (a->dup) job(0, a->dy, a->stride_dy, a->N, a->h, a->dup);
        if (a->ddown) job(1, a->x, a->stride_x, a->K, a->g, a->ddown);
        if (int rc = outer<T, RM>(a, g, j, s)) return rc;
        if (int rc = launch(lora_join_kernel<T>, dim3(joins[0].blocks + joins[1].blocks, a->A), 256, 0, 1, true, s, joins[0], joins[1])) return rc;
        g.chained = true;
    }
    if (a->dx) {
        g.x = nullptr; g.K = a->K; g.out = a->dx; g.stride_out = a->K; g.factor = a->down;
        return NB_TC_OR(a, tc_expand(g, true, a->dtype, s), (expand<T, RM, true>(g, s)));
    }
    return NB_OK;
}
template <typename T>
int dispatch(const nb_lora_args* a, bool backward, cudaStream_t s) {
    const int rm = a->R / 16;
    if (rm <= 1) return backward ? backward_t<T, 1>(a, s) : forward_t<T, 1>(a, s);
    if (rm <= 2) return backward ? backward_t<T, 2>(a, s) : forward_t<T, 2>(a, s);
    if (rm <= 4) return backward ? backward_t<T, 4>(a, s) : forward_t<T, 4>(a, s);
    return backward ? backward_t<T, 8>(a, s) : forward_t<T, 8>(a, s);
}

int check(const nb_lora_args* a) {
    NB_REQUIRE(a && a->T >= 0 && a->K > 0 && a->N > 0 && a->R > 0 && a->A > 0 && a->requests >= 0);
    NB_REQUIRE(a->dtype == NB_DTYPE_BF16 || a->dtype == NB_DTYPE_FP16);
    NB_REQUIRE(a->impl == NB_IMPL_AUTO || a->impl == NB_IMPL_TCGEN05 || a->impl == NB_IMPL_GENERIC);
    if (a->R % 16 || a->R > NB_LORA_MAX_RANK) return fail_with(NB_ERR_UNSUPPORTED, "the rank must be a multiple of 16 up to NB_LORA_MAX_RANK");
    if (a->K % 8 || a->N % 8) return fail_with(NB_ERR_UNSUPPORTED, "K and N must be multiples of 8");
    if (a->T > (1 << 30) || a->requests > 65535 || a->A > 65535 || item_count(a->T, a->requests, kRows) > 65535 || a->K > (1 << 24) || a->N > (1 << 24))
        return fail_with(NB_ERR_TOO_LARGE, "rows / 64 + requests or adapters above 65535, or more than 2^24 columns");
    if (a->T == 0) return NB_OK;
    NB_REQUIRE(a->offsets && (a->adapters || a->requests == 0) && a->down && a->up && aligned16(a->down) && aligned16(a->up));
    return NB_OK;
}

}  // namespace
}  // namespace lora
}  // namespace nb

extern "C" int64_t nb_lora_workspace_bytes(const nb_lora_args* a) {
    using namespace nb;
    using namespace nb::lora;
    if (check(a) != NB_OK || a->T == 0) return 0;
    int64_t bytes = 0;
    if (a->dup) bytes = piece_of(a, a->N, bytes).end;
    if (a->ddown) bytes = piece_of(a, a->K, bytes).end;
    return bytes;
}

extern "C" int64_t nb_lora_h_bytes(const nb_lora_args* a) {
    using namespace nb;
    using namespace nb::lora;
    if (!a || a->T < 0 || a->T > (1 << 30) || a->R <= 0 || a->R % 16 || a->R > NB_LORA_MAX_RANK) return 0;
    return (parts_of(a->dtype) * plane_bytes(a->T, a->R) + (scaled(a->dtype) ? 4ll * a->T : 0) + 15) / 16 * 16;
}

extern "C" int nb_lora_forward(const nb_lora_args* a, void* stream) {
    using namespace nb;
    using namespace nb::lora;
    if (int rc = check(a)) return rc;
    if (a->T == 0) return NB_OK;
    NB_REQUIRE(a->x && a->out && a->h && aligned16(a->x) && aligned16(a->out) && aligned16(a->h) && aligned16(a->base));
    NB_REQUIRE(a->stride_x % 8 == 0 && a->stride_out % 8 == 0 && (!a->base || a->stride_base % 8 == 0));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a->dtype == NB_DTYPE_BF16 ? dispatch<__nv_bfloat16>(a, false, s) : dispatch<__half>(a, false, s);
}

extern "C" int nb_lora_backward(const nb_lora_args* a, void* stream) {
    using namespace nb;
    using namespace nb::lora;
    if (int rc = check(a)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->T == 0) {  // empty sums
        if (a->ddown) NB_CUDA_CHECK(cudaMemsetAsync(a->ddown, 0, (size_t)a->A * a->R * a->K * 2, s));
        if (a->dup) NB_CUDA_CHECK(cudaMemsetAsync(a->dup, 0, (size_t)a->A * a->R * a->N * 2, s));
        return NB_OK;
    }
    if (!a->dx && !a->ddown && !a->dup) return NB_OK;
    NB_REQUIRE(a->dy && aligned16(a->dy) && a->stride_dy % 8 == 0);
    NB_REQUIRE(!(a->dx || a->ddown) || (a->g && aligned16(a->g)));
    NB_REQUIRE(!a->ddown || (a->x && aligned16(a->x) && a->stride_x % 8 == 0 && aligned16(a->ddown)));
    NB_REQUIRE(!a->dup || (a->h && aligned16(a->h) && aligned16(a->dup)));
    NB_REQUIRE(aligned16(a->dx));
    if (a->dup || a->ddown) {
        NB_REQUIRE(a->workspace && (reinterpret_cast<uintptr_t>(a->workspace) & 255) == 0);
        if (a->workspace_bytes < nb_lora_workspace_bytes(a)) return fail_with(NB_ERR_INVALID, "workspace smaller than nb_lora_workspace_bytes()");
    }
    return a->dtype == NB_DTYPE_BF16 ? dispatch<__nv_bfloat16>(a, true, s) : dispatch<__half>(a, true, s);
}
