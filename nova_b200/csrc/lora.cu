// Low-rank adapters of many requests beside a shared projection:
// out = base + s (x A^T) B^T, the rows of each adapter gathered into tiles.
//
// 2 r (K + N) flops per row against 2 K + 4 N bytes of it and 2 r (K + N) of
// its adapter: memory at any length, and for single tokens the latency of the
// chain x A^T -> h -> h B^T.  So one launch does both products: a cluster of 8
// CTAs takes a tile of up to 16 or 64 rows, each CTA an eighth of K for the
// first product; of the partial sums (rows x rank, fp32) each CTA adds an
// eighth, in CTA order, through distributed shared memory and hands the result
// to all, and each then has all of h for its eighth of N.  h is rounded to fp16 for the second product (2^-11
// of the adapter's term, which is added to base in fp32 before the one rounding
// of the result).  Fragments of mma.sync m16n8k16 are read straight from
// global memory: the contraction index is permuted so that a lane's operand
// registers are 16 (x, A) or 8 (B) consecutive bytes, and the columns of four
// neighbouring tiles are dealt so that a lane's results are 16 consecutive
// bytes of base and out.
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
    const int4* tiles;
    const int* rows;
    int k, n, max_rank, copy;    // copy: rows without an adapter are copied (out is not base)
};

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// RT: rank tiles of 8 (rank <= 8 RT).  MT: row tiles of 16.
template <int RT, int MT>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) lora_add_kernel(const Params p) {
    constexpr int R = 8 * RT, TM = 16 * MT, KS = WARPS / MT;   // KS warps share a row tile's part of K
    constexpr int HP = R + 8;                                  // padded row of h
    extern __shared__ __align__(16) uint8_t smem[];
    float* red = reinterpret_cast<float*>(smem);               // [KS][TM][R], then this CTA's sums in [0]
    __half* hs = reinterpret_cast<__half*>(red + KS * TM * R); // [TM][HP]
    __shared__ int row_of[TM];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int cr = int(blockIdx.x) % CLUSTER;
    pdl_wait();
    const int4 tile = p.tiles[blockIdx.x / CLUSTER];
    const int adapter = tile.x, rank = tile.y, count = tile.w;
    if (threadIdx.x < TM) row_of[threadIdx.x] = int(threadIdx.x) < count ? p.rows[tile.z + threadIdx.x] : -1;
    __syncthreads();
    const int n32 = (p.n + 31) / 32, nb0 = cr * n32 / CLUSTER, nb1 = (cr + 1) * n32 / CLUSTER;

    if (adapter < 0) {      // the whole cluster has this tile: nobody waits below
        if (p.copy)
            for (int r = warp; r < count; r += WARPS)
                for (int c = nb0 * 32 + lane * 8; c < min(nb1 * 32, p.n); c += 256)
                    *reinterpret_cast<uint4*>(p.out + row_of[r] * p.out_stride + c) =
                        *reinterpret_cast<const uint4*>(p.base + row_of[r] * p.base_stride + c);
        return;
    }

    // ---- h = x A^T over this CTA's part of K
    const int mt = warp % MT, ks = warp / MT;
    {
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
        for (int c = k0 + ks; c < k1; c += KS) {
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
        float* dst = red + (ks * TM + mt * 16) * R;
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            *reinterpret_cast<float2*>(dst + g * R + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(dst + (g + 8) * R + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TM * R; i += THREADS) {
        float s = red[i];
#pragma unroll
        for (int w = 1; w < KS; ++w) s += red[w * TM * R + i];
        red[i] = s;
    }
    // ---- out = base + h B^T over this CTA's part of N: 32 columns a warp, B read once for all rows of the tile.
    // What the first product does not change is requested now, so that it arrives during the exchange.
    constexpr int S = RT / 2;                // steps of 16 along the rank
    const __half* bw = p.b + int64_t(adapter) * p.n * p.max_rank + 4 * t;
    uint4 ba[MT], bb[MT];
    uint2 w[4][S];
    auto load = [&](int nb) {
        const int n0 = nb * 32, col = n0 + 8 * t;
        const bool in = col < p.n;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int ra = row_of[m * 16 + g], rb = row_of[m * 16 + g + 8];
            ba[m] = in && ra >= 0 ? *reinterpret_cast<const uint4*>(p.base + ra * p.base_stride + col) : zero4();
            bb[m] = in && rb >= 0 ? *reinterpret_cast<const uint4*>(p.base + rb * p.base_stride + col) : zero4();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                w[j][s] = make_uint2(0u, 0u);
                if (rank > 16 * s + 4 * t && c < p.n) w[j][s] = *reinterpret_cast<const uint2*>(bw + int64_t(c) * p.max_rank + 16 * s);
            }
        }
    };
    int nb = nb0 + warp;
    if (nb < nb1) load(nb);

    // ---- the clusters' partial sums: CTA i adds the i-th eighth of h, in CTA order, and hands it to every CTA
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const float scale = p.scaling ? p.scaling[adapter] : 1.f;
    constexpr int SHARE = TM * R / CLUSTER / 2;      // pairs of elements
    for (int i = threadIdx.x; i < SHARE; i += THREADS) {
        const int at = cr * SHARE + i;
        float2 v[CLUSTER];
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k) v[k] = reinterpret_cast<const float2*>(cluster.map_shared_rank(red, k))[at];
        float2 s = v[0];
#pragma unroll
        for (int k = 1; k < CLUSTER; ++k) s = make_float2(s.x + v[k].x, s.y + v[k].y);
        const __half2 h = __floats2half2_rn(s.x * scale, s.y * scale);
        const int off = (2 * at / R) * HP + 2 * at % R;
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k) *reinterpret_cast<__half2*>(cluster.map_shared_rank(hs, k) + off) = h;
    }
    cluster.sync();                          // h is complete everywhere; no CTA reads or writes another's memory from here

    for (; nb < nb1; nb += WARPS) {
        const int col = nb * 32 + 8 * t;
        const bool in = col < p.n;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int left = rank - (16 * s + 4 * t);          // entries of this rank that the lane's four hold
            if (left >= 4) continue;
            const uint32_t mx = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u, my = left == 3 ? 0xFFFFu : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j][s].x &= mx;
                w[j][s].y &= my;
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const uint2 lo = *reinterpret_cast<const uint2*>(hs + (m * 16 + g) * HP + 16 * s + 4 * t);
                const uint2 hi = *reinterpret_cast<const uint2*>(hs + (m * 16 + g + 8) * HP + 16 * s + 4 * t);
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_16816(acc[j], lo.x, hi.x, lo.y, hi.y, w[j][s].x, w[j][s].y);
            }
            const uint32_t wa[4] = {ba[m].x, ba[m].y, ba[m].z, ba[m].w}, wb[4] = {bb[m].x, bb[m].y, bb[m].z, bb[m].w};
            uint32_t oa[4], ob[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&wa[j]));
                const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&wb[j]));
                oa[j] = pack_f16x2(fa.x + acc[j][0], fa.y + acc[j][1]);
                ob[j] = pack_f16x2(fb.x + acc[j][2], fb.y + acc[j][3]);
            }
            const int ra = row_of[m * 16 + g], rb = row_of[m * 16 + g + 8];
            if (in && ra >= 0) *reinterpret_cast<uint4*>(p.out + ra * p.out_stride + col) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
            if (in && rb >= 0) *reinterpret_cast<uint4*>(p.out + rb * p.out_stride + col) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
        }
        if (nb + WARPS < nb1) load(nb + WARPS);
    }
}

template <int RT, int MT>
int run(const Params& p, int64_t tiles, cudaStream_t stream) {
    constexpr int R = 8 * RT, TM = 16 * MT, KS = WARPS / MT;
    constexpr int bytes = KS * TM * R * 4 + TM * (R + 8) * 2;
    static bool ready[kMaxDevices];        // shared-memory limit raised on this device
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices || !ready[dev]) {
        if (cudaFuncSetAttribute(reinterpret_cast<const void*>(&lora_add_kernel<RT, MT>),
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
            return check_launch("lora add");
        if (dev >= 0 && dev < kMaxDevices) ready[dev] = true;
    }
    launch(lora_add_kernel<RT, MT>, dim3(unsigned(tiles * CLUSTER)), dim3(THREADS), bytes, stream, p);
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
    if (!a->base || !a->out || !a->tiles || !a->rows || (a->adapters && (!a->x || !a->a || !a->b)))
        return fail(NOVA_ERR_INVALID, "lora add: NULL pointer");
    if (a->x_stride < a->k || a->base_stride < a->n || a->out_stride < a->n)
        return fail(NOVA_ERR_INVALID, "lora add: row strides below the row length");
    auto off = [](const void* p, int64_t al) { return reinterpret_cast<uintptr_t>(p) % al != 0; };
    if (off(a->x, 16) || off(a->base, 16) || off(a->out, 16) || off(a->a, 16) || off(a->b, 16) || off(a->tiles, 16) ||
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
    p.tiles = reinterpret_cast<const int4*>(a->tiles);
    p.rows = a->rows;
    p.k = int(a->k);
    p.n = int(a->n);
    p.max_rank = int(a->max_rank);
    p.copy = a->out != a->base;
    const int rt = a->max_rank <= 16 ? 2 : a->max_rank <= 32 ? 4 : a->max_rank <= 64 ? 8 : 16;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->tile_rows == 16)
        return rt == 2 ? run<2, 1>(p, a->n_tiles, s) : rt == 4 ? run<4, 1>(p, a->n_tiles, s)
             : rt == 8 ? run<8, 1>(p, a->n_tiles, s) : run<16, 1>(p, a->n_tiles, s);
    return rt == 2 ? run<2, 4>(p, a->n_tiles, s) : rt == 4 ? run<4, 4>(p, a->n_tiles, s)
         : rt == 8 ? run<8, 4>(p, a->n_tiles, s) : run<16, 4>(p, a->n_tiles, s);
}
