// Low-rank adapters of many requests beside a shared projection:
// out = base + s (x A^T) B^T, the rows of each adapter gathered into tiles.
//
// 2 r (K + N) flops per row against 2 K + 4 N bytes of it and 2 r (K + N) of
// its adapter: memory at any length, and for single tokens the latency of the
// chain x A^T -> h -> h B^T.  The first product is split over K between the 8
// CTAs of a cluster, whose partial sums (rows x rank, fp32) meet in distributed
// shared memory and are added in CTA order.  h is rounded to fp16 for the second
// product: each row is first multiplied by the power of two that brings its
// largest entry to [2^14, 2^15), and that power and the adapter's scaling go on
// the fp32 sums of the second product.  So the error is 2^-11 of the sum of
// |s h_j B_j| at any size of x, A and s (entries 2^-28 below the row's largest
// lose bits), and the result is rounded once, with base.
//   * few rows (16-row tiles): one launch; each CTA goes on with an eighth of N;
//   * many (64-row tiles): h goes through memory and a second launch takes the
//     columns.  As one launch a cluster held its 8 CTAs for the whole of N, and
//     37 of them did not fit the GPU at once: 93 us against 69 for 2217 rows (1750
//     of them with an adapter) of 19456 columns at rank 64.  It is 71.5 since h's
//     rows have powers of their own (16 us for the first product, 54 for the second:
//     144 MB of DRAM traffic, 22 us of it, and 20 us of mma.sync).
// 64 rows with 24 adapters of rank up to 16, 2560 -> 6144: one launch, 8.2 us a
// call, 9.7 of kernel with cold caches.
// Fragments of mma.sync m16n8k16 are read straight from global memory: the
// contraction index is permuted so that a lane's operand registers are 16
// consecutive bytes (8 of B and h at rank 16), and the columns of four neighbouring tiles are
// dealt so that a lane's results are 16 consecutive bytes of base and out.
#include <cooperative_groups.h>

#include "common.cuh"

namespace nova {
namespace lora {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;
constexpr int WARPS = 8;
constexpr int CLUSTER = 8;

struct Params {
    const __half* x;
    int64_t x_stride;
    const __half* base;
    int64_t base_stride;
    __half* out;
    int64_t out_stride;
    const __half* a;
    const __half* b;
    const float* scaling;
    const int* tiles;            // per tile: adapter, rank, rows, 0, then the rows (padded to the tile with -1)
    __half* h;                   // 64-row tiles: the first product, [tile][64][R]
    float* factor;               // and what its rows are to be multiplied by, [tile][64]
    int k, n, max_rank, copy;    // copy: rows without an adapter are copied (out is not base)
};

// The rank that the kernels are built for: what h has room for.
inline int64_t rank_tile(int64_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }
// h and its rows' factors of 64-row tiles.
inline int64_t h_bytes(int64_t tiles, int64_t r) { return tiles * 64 * r * 2; }
inline int64_t workspace_bytes(int64_t tiles, int64_t r) { return h_bytes(tiles, r) + tiles * 64 * 4; }

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// RT: rank tiles of 8 (rank <= 8 RT).  MT: row tiles of 16.
template <int RT, int MT>
struct Shape {
    static constexpr int R = 8 * RT, TM = 16 * MT, KS = WARPS / MT;   // KS warps share a row tile's part of K
    static constexpr int HP = R == 16 ? 32 : R == 32 ? 32 : R + 32;   // padded row of h: its reads hit all banks
    static constexpr int RED = KS * TM * R * 4, H = TM * HP * 2;      // bytes of partial sums, of h
};

// This CTA's part of x A^T for a tile, fp32 sums over its warps in red[0 .. TM * R).
template <int RT, int MT>
__device__ __forceinline__ void shrink(const Params& p, int adapter, int rank, const int* row_of, float* red, int cr) {
    using S = Shape<RT, MT>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int mt = warp % MT, ks = warp / MT;
    const int nk = (p.k + 31) / 32;
    const int k0 = cr * nk / CLUSTER, k1 = (cr + 1) * nk / CLUSTER;
    const int ra = row_of[mt * 16 + g], rb = row_of[mt * 16 + g + 8];
    const __half* xa = ra >= 0 ? p.x + ra * p.x_stride + 8 * t : nullptr;
    const __half* xb = rb >= 0 ? p.x + rb * p.x_stride + 8 * t : nullptr;
    const __half* aw = p.a + int64_t(adapter) * p.max_rank * p.k + 8 * t;
    float acc[RT][4];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    constexpr int U = RT <= 2 ? 4 : RT <= 8 ? 2 : 1;   // 128 registers hold so many chunks in flight
#pragma unroll U
    for (int c = k0 + ks; c < k1; c += S::KS) {
        const int k = c * 32;
        const bool in = k + 8 * t < p.k;
        const uint4 va = in && xa ? *reinterpret_cast<const uint4*>(xa + k) : zero4();
        const uint4 vb = in && xb ? *reinterpret_cast<const uint4*>(xb + k) : zero4();
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const uint4 w = in && 8 * j + g < rank ? *reinterpret_cast<const uint4*>(aw + int64_t(8 * j + g) * p.k + k) : zero4();
            mma_16816(acc[j], va.x, vb.x, va.y, vb.y, w.x, w.y);
            mma_16816(acc[j], va.z, vb.z, va.w, vb.w, w.z, w.w);
        }
    }
    float* dst = red + (ks * S::TM + mt * 16) * S::R;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        *reinterpret_cast<float2*>(dst + g * S::R + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(dst + (g + 8) * S::R + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < S::TM * S::R; i += THREADS) {
        float v = red[i];
#pragma unroll
        for (int w = 1; w < S::KS; ++w) v += red[w * S::TM * S::R + i];
        red[i] = v;
    }
}

// What a row of h is multiplied by before it is rounded to fp16, and what undoes
// it: the powers of two that bring its largest magnitude to [2^14, 2^15).  A sum
// of products of fp16 numbers is a multiple of 2^-48 below 2^63; a row of zeros
// takes the clamped power, and one that is not finite stays so.
struct Power {
    float to, back;
};
__device__ __forceinline__ Power row_power(float largest) {
    const int e = max(int(__float_as_uint(largest) >> 23) - 127, -100);
    return {__uint_as_float(uint32_t(127 + 14 - e) << 23), __uint_as_float(uint32_t(127 + e - 14) << 23)};
}
// Largest of N consecutive lanes, in all of them.
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int off = N / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}

// CTA i of the cluster adds the i-th eighth of h over all CTAs, in CTA order, a
// warp one row: fp16 rows to h_out, what they are to be multiplied by to f_out.
template <int RT>
__device__ __forceinline__ void gather(cg::cluster_group& cluster, float* red, int cr, float scale, __half* h_out, float* f_out) {
    using S = Shape<RT, 4>;
    static_assert(S::TM / CLUSTER == WARPS, "a row of h per warp");
    constexpr int N = (S::R / 2 + 31) / 32;                    // pairs per lane
    const int row = cr * WARPS + int(threadIdx.x >> 5), lane = threadIdx.x & 31;
    float2 s[N];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = min(lane + 32 * i, S::R / 2 - 1);       // ranks up to 32: the last pair again
        float2 v[CLUSTER];
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k)
            v[k] = reinterpret_cast<const float2*>(cluster.map_shared_rank(red, k))[row * (S::R / 2) + at];
        s[i] = v[0];
#pragma unroll
        for (int k = 1; k < CLUSTER; ++k) s[i] = make_float2(s[i].x + v[k].x, s[i].y + v[k].y);
        top = fmaxf(top, fmaxf(fabsf(s[i].x), fabsf(s[i].y)));
    }
    const Power pw = row_power(lanes_max<32>(top));
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane + 32 * i < S::R / 2)
            *reinterpret_cast<__half2*>(h_out + row * S::R + 2 * (lane + 32 * i)) = __floats2half2_rn(s[i].x * pw.to, s[i].y * pw.to);
    if (lane == 0) f_out[row] = pw.back * scale;
}

// 32 columns of the second product for MW row tiles of 16, B in registers once.
template <int RT, int MW>
struct Columns {
    static constexpr int S = RT / 2;           // steps of 16 along the rank
    uint4 ba[MW], bb[MW];
    uint2 w[4][S];

    // The lane's first of the four entries along the rank that it holds in step s: two steps' are neighbours, so that
    // they come in one load of 16 bytes (2217 rows of 19456 columns at rank 64, h then unscaled: 70.2 us with loads of
    // 8, 68.4 with 16).
    static __device__ __forceinline__ int entry(int s, int t) { return S == 1 ? 4 * t : 32 * (s / 2) + 8 * t + 4 * (s % 2); }
    // Those entries of every step, `n` of them to be read at `p`.
    static __device__ __forceinline__ void entries(const __half* p, int n, int t, uint2 (&v)[S]) {
        if constexpr (S == 1) {
            v[0] = 4 * t < n ? *reinterpret_cast<const uint2*>(p + 4 * t) : make_uint2(0u, 0u);
        } else {
#pragma unroll
            for (int s = 0; s < S; s += 2) {
                const uint4 q = entry(s, t) < n ? *reinterpret_cast<const uint4*>(p + entry(s, t)) : zero4();
                v[s] = make_uint2(q.x, q.y);
                v[s + 1] = make_uint2(q.z, q.w);
            }
        }
    }

    __device__ __forceinline__ void load(const Params& p, const __half* bw, int rank, const int* row_of, int nb, int g, int t) {
        const int n0 = nb * 32, col = n0 + 8 * t;
        const bool in = col < p.n;
#pragma unroll
        for (int m = 0; m < MW; ++m) {
            const int ra = row_of[m * 16 + g], rb = row_of[m * 16 + g + 8];
            ba[m] = in && ra >= 0 ? *reinterpret_cast<const uint4*>(p.base + ra * p.base_stride + col) : zero4();
            bb[m] = in && rb >= 0 ? *reinterpret_cast<const uint4*>(p.base + rb * p.base_stride + col) : zero4();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
            entries(bw + int64_t(c) * p.max_rank, c < p.n ? rank : 0, t, w[j]);
        }
    }

    // hs: the first row tile's h, rows of hp elements; factor: what each row of the product is multiplied by.
    __device__ __forceinline__ void finish(const Params& p, const __half* hs, int hp, const float* factor, int rank,
                                           const int* row_of, int nb, int g, int t) {
        const int col = nb * 32 + 8 * t;
        const bool in = col < p.n;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int left = rank - entry(s, t);               // entries of this rank that the lane's four hold
            if (left >= 4) continue;
            const uint32_t mx = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u, my = left == 3 ? 0xFFFFu : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j][s].x &= mx;
                w[j][s].y &= my;
            }
        }
#pragma unroll
        for (int m = 0; m < MW; ++m) {
            const float xa = factor[m * 16 + g], xb = factor[m * 16 + g + 8];
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
            for (int s = 0; s < S; s += 2) {
                uint4 lo, hi;
                if constexpr (S == 1) {
                    const uint2 a = *reinterpret_cast<const uint2*>(hs + (m * 16 + g) * hp + 4 * t);
                    const uint2 b = *reinterpret_cast<const uint2*>(hs + (m * 16 + g + 8) * hp + 4 * t);
                    lo = make_uint4(a.x, a.y, 0u, 0u);
                    hi = make_uint4(b.x, b.y, 0u, 0u);
                } else {
                    lo = *reinterpret_cast<const uint4*>(hs + (m * 16 + g) * hp + entry(s, t));
                    hi = *reinterpret_cast<const uint4*>(hs + (m * 16 + g + 8) * hp + entry(s, t));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma_16816(acc[j], lo.x, hi.x, lo.y, hi.y, w[j][s].x, w[j][s].y);
                    if constexpr (S > 1) mma_16816(acc[j], lo.z, hi.z, lo.w, hi.w, w[j][s + 1].x, w[j][s + 1].y);
                }
            }
            const uint32_t wa[4] = {ba[m].x, ba[m].y, ba[m].z, ba[m].w}, wb[4] = {bb[m].x, bb[m].y, bb[m].z, bb[m].w};
            uint32_t oa[4], ob[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&wa[j]));
                const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&wb[j]));
                oa[j] = pack_f16x2(fmaf(acc[j][0], xa, fa.x), fmaf(acc[j][1], xa, fa.y));
                ob[j] = pack_f16x2(fmaf(acc[j][2], xb, fb.x), fmaf(acc[j][3], xb, fb.y));
            }
            const int ra = row_of[m * 16 + g], rb = row_of[m * 16 + g + 8];
            if (in && ra >= 0) *reinterpret_cast<uint4*>(p.out + ra * p.out_stride + col) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
            if (in && rb >= 0) *reinterpret_cast<uint4*>(p.out + rb * p.out_stride + col) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
        }
    }
};

// Columns [c0, c1) of the rows without an adapter.
__device__ __forceinline__ void copy_rows(const Params& p, const int* row_of, int count, int c0, int c1) {
    for (int r = threadIdx.x >> 5; r < count; r += WARPS)
        for (int c = c0 + int(threadIdx.x & 31) * 8; c < min(c1, p.n); c += 256)
            *reinterpret_cast<uint4*>(p.out + row_of[r] * p.out_stride + c) =
                *reinterpret_cast<const uint4*>(p.base + row_of[r] * p.base_stride + c);
}

struct Tile {
    int adapter, rank, count;
};
__device__ __forceinline__ Tile read_tile(const Params& p, int tile, int tm, int* row_of) {
    const int* rec = p.tiles + int64_t(tile) * (4 + tm);
    if (int(threadIdx.x) < tm) row_of[threadIdx.x] = rec[4 + threadIdx.x];
    const int4 head = *reinterpret_cast<const int4*>(rec);
    __syncthreads();
    return {head.x, head.y, head.z};
}

// Both products of a 16-row tile in one launch (single tokens, few rows).  Every
// CTA pushes its sums to all CTAs of the cluster, and each adds them up for
// itself: one cluster barrier between the products, no remote load.
template <int RT>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) lora_add_kernel(const Params p) {
    using S = Shape<RT, 1>;
    constexpr int E = S::TM * S::R;                            // elements of h
    extern __shared__ __align__(16) uint8_t smem[];
    float* red = reinterpret_cast<float*>(smem);               // [KS][E], this CTA's sums in [0]
    float* from = reinterpret_cast<float*>(smem + S::RED);     // [CLUSTER][E]
    __half* hs = reinterpret_cast<__half*>(smem + S::RED + CLUSTER * E * 4);
    __shared__ int row_of[S::TM];
    __shared__ float factor[S::TM];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cr = int(blockIdx.x) % CLUSTER;
    pdl_wait();
    const Tile tile = read_tile(p, blockIdx.x / CLUSTER, S::TM, row_of);
    const int n32 = (p.n + 31) / 32, nb0 = cr * n32 / CLUSTER, nb1 = (cr + 1) * n32 / CLUSTER;
    if (tile.adapter < 0) { // the whole cluster has this tile: nobody waits below
        if (p.copy) copy_rows(p, row_of, tile.count, nb0 * 32, nb1 * 32);
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();                                  // this CTA runs: the others may write to it
    shrink<RT, 1>(p, tile.adapter, tile.rank, row_of, red, cr);
    // what the first product does not change is requested now, so that it arrives during the exchange
    const __half* bw = p.b + int64_t(tile.adapter) * p.n * p.max_rank;
    constexpr int AHEAD = RT <= 2 ? 3 : RT <= 4 ? 2 : 1;       // 32-column groups that registers hold
    Columns<RT, 1> c[AHEAD];
    int nb = nb0 + warp;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (nb + i * WARPS < nb1) c[i].load(p, bw, tile.rank, row_of, nb + i * WARPS, g, t);
    const float scale = p.scaling ? p.scaling[tile.adapter] : 1.f;
    cluster.barrier_wait();
    for (int i = threadIdx.x; i < E; i += THREADS) {           // the element that this thread has summed
        const float v = red[i];
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k) cluster.map_shared_rank(from, k)[cr * E + i] = v;
    }
    cluster.sync();         // every CTA's sums are here; no CTA touches another's memory from now on
    // a warp adds up two rows: lanes 0-15 and 16-31 one each at rank 16, all lanes one after the other above
    constexpr int N = 2 * S::R / 32, PER = S::R <= 32 ? 1 : S::R / 32;   // elements per lane; of one row
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = warp * 2 * S::R + 32 * i + lane;
        v[i] = from[at];
#pragma unroll
        for (int k = 1; k < CLUSTER; ++k) v[i] += from[k * E + at];
    }
#pragma unroll
    for (int i = 0; i < N; i += PER) {
        float top = fabsf(v[i]);
#pragma unroll
        for (int j = 1; j < PER; ++j) top = fmaxf(top, fabsf(v[i + j]));
        const Power pw = row_power(lanes_max<(S::R < 32 ? S::R : 32)>(top));
        const int row = (warp * 2 * S::R + 32 * i + lane) / S::R;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            hs[row * S::HP + (32 * (i + j) + lane) % S::R] = __float2half_rn(v[i + j] * pw.to);
        if (lane % (S::R < 32 ? S::R : 32) == 0) factor[row] = pw.back * scale;
    }
    __syncthreads();
    for (; nb < nb1; nb += AHEAD * WARPS) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int at = nb + i * WARPS, later = at + AHEAD * WARPS;
            if (at < nb1) c[i].finish(p, hs, S::HP, factor, tile.rank, row_of, at, g, t);
            if (later < nb1) c[i].load(p, bw, tile.rank, row_of, later, g, t);
        }
    }
}

// The first product of 64-row tiles -> h (fp16 [tile][64][R]) and its rows' factors in the workspace.
template <int RT>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) lora_shrink_kernel(const Params p) {
    using S = Shape<RT, 4>;
    extern __shared__ __align__(16) uint8_t smem[];
    float* red = reinterpret_cast<float*>(smem);
    __shared__ int row_of[S::TM];
    const int cr = int(blockIdx.x) % CLUSTER, at = blockIdx.x / CLUSTER;
    pdl_wait();
    const Tile tile = read_tile(p, at, S::TM, row_of);
    if (tile.adapter < 0) return;
    shrink<RT, 4>(p, tile.adapter, tile.rank, row_of, red, cr);
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    gather<RT>(cluster, red, cr, p.scaling ? p.scaling[tile.adapter] : 1.f, p.h + int64_t(at) * S::TM * S::R,
               p.factor + int64_t(at) * S::TM);
    cluster.sync();         // the others have read this CTA's sums
}

// The second product of 64-row tiles: COLS columns of a tile per CTA, a warp 32
// rows x 32 columns at a time.
constexpr int COLS = 512;

template <int RT>
__global__ void __launch_bounds__(THREADS, RT <= 4 ? 3 : 2) lora_expand_kernel(const Params p) {
    using S = Shape<RT, 4>;
    __shared__ __align__(16) __half hs[S::TM * S::HP];
    __shared__ int row_of[S::TM];
    __shared__ float factor[S::TM];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    const Tile tile = read_tile(p, blockIdx.y, S::TM, row_of);
    const int c0 = int(blockIdx.x) * COLS, c1 = min(c0 + COLS, p.n);
    if (tile.adapter < 0) {
        if (p.copy) copy_rows(p, row_of, tile.count, c0, c1);
        return;
    }
    const int* rows = row_of + (warp & 1) * 32;
    const __half* bw = p.b + int64_t(tile.adapter) * p.n * p.max_rank;
    Columns<RT, 2> c;
    int nb = c0 / 32 + (warp >> 1);
    const int nb1 = (c1 + 31) / 32;
    if (nb < nb1) c.load(p, bw, tile.rank, rows, nb, g, t);
    const uint4* h_in = reinterpret_cast<const uint4*>(p.h + int64_t(blockIdx.y) * S::TM * S::R);
    for (int i = threadIdx.x; i < S::TM * S::R / 8; i += THREADS)
        *reinterpret_cast<uint4*>(hs + i / RT * S::HP + i % RT * 8) = h_in[i];
    if (threadIdx.x < S::TM) factor[threadIdx.x] = p.factor[int64_t(blockIdx.y) * S::TM + threadIdx.x];
    __syncthreads();
    for (; nb < nb1; nb += WARPS / 2) {
        c.finish(p, hs + (warp & 1) * 32 * S::HP, S::HP, factor + (warp & 1) * 32, tile.rank, rows, nb, g, t);
        if (nb + WARPS / 2 < nb1) c.load(p, bw, tile.rank, rows, nb + WARPS / 2, g, t);
    }
}

// Raises a kernel's shared-memory limit, once per device.
template <typename K>
int allow_smem(K kernel, int bytes, bool (&ready)[kMaxDevices]) {
    const int dev = current_device();
    if (dev >= 0 && dev < kMaxDevices && ready[dev]) return NOVA_OK;
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
        return check_launch("lora add");
    if (dev >= 0 && dev < kMaxDevices) ready[dev] = true;
    return NOVA_OK;
}

template <int RT>
int run(const Params& p, int64_t tiles, bool wide, cudaStream_t stream) {
    static bool ready[2][kMaxDevices];
    const dim3 grid(unsigned(tiles * CLUSTER)), block(THREADS);
    if (!wide) {
        constexpr int bytes = Shape<RT, 1>::RED + CLUSTER * 16 * 8 * RT * 4 + Shape<RT, 1>::H;
        if (int rc = allow_smem(&lora_add_kernel<RT>, bytes, ready[0])) return rc;
        launch(lora_add_kernel<RT>, grid, block, bytes, stream, p);
        return check_launch("lora add");
    }
    constexpr int bytes = Shape<RT, 4>::RED;
    if (int rc = allow_smem(&lora_shrink_kernel<RT>, bytes, ready[1])) return rc;
    launch(lora_shrink_kernel<RT>, grid, block, bytes, stream, p);
    if (int rc = check_launch("lora add")) return rc;
    launch(lora_expand_kernel<RT>, dim3(unsigned((p.n + COLS - 1) / COLS), unsigned(tiles)), block, 0, stream, p);
    return check_launch("lora add");
}

}  // namespace lora
}  // namespace nova

using namespace nova;

extern "C" int nova_lora_add(const nova_lora_args* a, void* stream) {
    using namespace nova::lora;
    if (!a) return fail(NOVA_ERR_INVALID, "lora add: args must not be NULL");
    if (a->n_tiles < 0 || a->tokens < 0 || a->n_tiles >= (1ll << 27) || a->tokens >= (1ll << 31))
        return fail(NOVA_ERR_INVALID, "lora add: tiles=%lld, tokens=%lld", (long long)a->n_tiles, (long long)a->tokens);
    if (!a->n_tiles) return NOVA_OK;
    if (a->tile_rows != 16 && a->tile_rows != 64) return fail(NOVA_ERR_INVALID, "lora add: tile_rows must be 16 or 64");
    if (a->k < 8 || a->n < 8 || a->k % 8 || a->n % 8 || a->k >= (1ll << 30) || a->n >= (1ll << 30))
        return fail(NOVA_ERR_INVALID, "lora add: k=%lld and n=%lld must be multiples of 8", (long long)a->k, (long long)a->n);
    if (a->adapters < 0 || (a->adapters && (a->max_rank < 8 || a->max_rank % 8 || a->max_rank > 128)))
        return fail(NOVA_ERR_UNSUPPORTED, "lora add: max_rank %lld must be a multiple of 8 up to 128", (long long)a->max_rank);
    if (a->top_rank < 0 || a->top_rank > a->max_rank)
        return fail(NOVA_ERR_INVALID, "lora add: top_rank %lld above max_rank %lld", (long long)a->top_rank, (long long)a->max_rank);
    if (!a->base || !a->out || !a->tiles || (a->adapters && (!a->x || !a->a || !a->b)))
        return fail(NOVA_ERR_INVALID, "lora add: NULL pointer");
    if (a->x_stride < a->k || a->base_stride < a->n || a->out_stride < a->n)
        return fail(NOVA_ERR_INVALID, "lora add: row strides below the row length");
    auto off = [](const void* p, int64_t al) { return reinterpret_cast<uintptr_t>(p) % al != 0; };
    if (off(a->x, 16) || off(a->base, 16) || off(a->out, 16) || off(a->a, 16) || off(a->b, 16) || off(a->tiles, 16) || off(a->workspace, 16) ||
        a->x_stride % 8 || a->base_stride % 8 || a->out_stride % 8)
        return fail(NOVA_ERR_ALIGN, "lora add: pointers need 16-byte alignment, strides multiples of 8");
    Params p{};
    p.x = static_cast<const __half*>(a->x);
    p.x_stride = a->x_stride;
    p.base = static_cast<const __half*>(a->base);
    p.base_stride = a->base_stride;
    p.out = static_cast<__half*>(a->out);
    p.out_stride = a->out_stride;
    p.a = static_cast<const __half*>(a->a);
    p.b = static_cast<const __half*>(a->b);
    p.scaling = static_cast<const float*>(a->scaling);
    p.tiles = a->tiles;
    p.k = int(a->k);
    p.n = int(a->n);
    p.max_rank = int(a->max_rank);
    p.copy = a->out != a->base;
    p.h = static_cast<__half*>(a->workspace);
    const bool wide = a->tile_rows == 64;
    const int64_t r = rank_tile(a->top_rank);
    if (wide && a->adapters && (!a->workspace || a->workspace_bytes < workspace_bytes(a->n_tiles, r)))
        return fail(NOVA_ERR_INVALID, "lora add: workspace of %lld bytes, %lld are needed", (long long)a->workspace_bytes,
                    (long long)workspace_bytes(a->n_tiles, r));
    p.factor = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + h_bytes(a->n_tiles, r));
    if (wide && a->n_tiles > 65535) return fail(NOVA_ERR_UNSUPPORTED, "lora add: %lld tiles", (long long)a->n_tiles);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return r == 16 ? run<2>(p, a->n_tiles, wide, s) : r == 32 ? run<4>(p, a->n_tiles, wide, s)
         : r == 64 ? run<8>(p, a->n_tiles, wide, s) : run<16>(p, a->n_tiles, wide, s);
}

extern "C" int nova_lora_workspace_bytes(int64_t n_tiles, int64_t tile_rows, int64_t top_rank, int64_t* bytes) {
    if (!bytes || n_tiles < 0 || top_rank < 0 || top_rank > 128)
        return fail(NOVA_ERR_INVALID, "lora workspace: tiles=%lld, top_rank=%lld", (long long)n_tiles, (long long)top_rank);
    *bytes = tile_rows == 64 ? lora::workspace_bytes(n_tiles, lora::rank_tile(top_rank)) : 0;
    return NOVA_OK;
}
