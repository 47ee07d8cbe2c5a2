// Attention of few query rows over the paged int8 cache (single tokens, a few
// speculated ones): o = sum_j softmax(q . k_j) v_j with the running maximum and
// sum, one pass over the cache.
//
// What bounds it is the cache: 272 bytes per token and KV head against 4 * 128
// flops per query row.  One CTA = (work item, KV head): a range of 64-token
// blocks of one request and up to 16 rows (token, query head) of that KV head,
// which share every K and V fragment.  Four warps each walk their own blocks
// with a private 17 KiB shared-memory stage; a page's K and V codes (one 128 x
// 128-byte TMA box, two halves) and scales (bulk copies) are requested per
// half, so that the next page's K loads while this page's V is used and the
// other way round.  Codes become fp16(code * step + min) in registers (byte
// permute, subtract 1024, one FMA) directly in the layout of an mma.sync A
// operand: S^T = K Q^T, O^T += V^T P^T, tokens and channels permuted so that
// every shared-memory read is 16 bytes and conflict-free.  P is transposed
// between the two products by movmatrix.  A tile's splits are joined in split
// order by the CTA that arrives last.  Measured: 32 requests of 8000 to 32768
// tokens with 8 KV heads, 1.26 GB, 213 us alone and 231 in a row (5.9 and 5.5
// TB/s); 16 requests of 40 to 8191, 70 MB, 20 us (the items are about three
// pages deep per warp: latency); one request of 77 tokens 5.2 us.
#include "paged.cuh"

namespace nova {
namespace paged {

int check_cache(const char* what, const void* codes, const void* scales, const void* tails, int64_t num_pages,
                int64_t num_tails, const void* plan, const nova_paged_plan_info* info);

int launch_tiles(const nova_paged_attn_args* a, const nova_paged_plan_info* info, const nova_paged_schedule& s,
                 cudaStream_t stream);

namespace rows {

constexpr int NW = 4;
constexpr int THREADS = NW * 32;
constexpr int STAGE = 17408;               // K codes, V codes, K min, K step, V min, V step of one page and head
constexpr int SC = 16384;
constexpr int TX_HALF = 8192 + 512;
constexpr int SMEM = NW * STAGE + 1024;

struct Params {
    const __half* q;
    int64_t q_t, q_h;
    const __half* scales;
    const __half* tails;
    __half* out;
    int64_t o_t, o_h;
    float* lse;
    const int* pages;
    const RowsItem* items;
    int* err;
    unsigned* counters;
    float* part;
    int q_heads, kv_heads, gq, window, tile_rows;
    float scale_log2;
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// Running maximum and sum of the NC columns (query rows) that this lane holds,
// updated with scores of T tokens each; x becomes the unnormalised weights.
// Rows that have seen no key keep m = -inf and weights of zero.
template <int NC, int T>
__device__ __forceinline__ void softmax_step(float (&x)[NC][T], float (&m)[NC], float (&l)[NC], float (&alpha)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float t = x[c][0];
#pragma unroll
        for (int i = 1; i < T; ++i) t = fmaxf(t, x[c][i]);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        const float m_new = fmaxf(m[c], t);
        const float base = m_new == -INFINITY ? 0.f : m_new;
        alpha[c] = exp2f(m[c] - base);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            x[c][i] = exp2f(x[c][i] - base);
            sum += x[c][i];
        }
        l[c] = l[c] * alpha[c] + sum;
        m[c] = m_new;
    }
}

// HL (at most 4 rows, one column tile): columns 4..7 repeat rows 0..3 and carry
// the low part of each weight, so P keeps ~22 bits at no cost.  Otherwise a
// column is a row and P is fp16: its rounding (2^-12 on average) averages out
// over the keys and is at most that of the fp16 output.
template <bool HL>
__device__ __forceinline__ uint32_t pack_p(float a, float b, int t) {
    if (HL && t >= 2) {
        a -= __half2float(__float2half_rn(a));
        b -= __half2float(__float2half_rn(b));
    }
    return pack_f16x2(a, b);
}

template <int NT, bool HL>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 3 : 2)
    paged_attn_rows_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tm) {
    constexpr int NC = 2 * NT;             // columns per lane: 8 n + 2t, 8 n + 2t + 1
    constexpr int RT = HL ? 4 : 8 * NT;    // rows per tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t bars[2][NW];
    __shared__ float sm_m[NW][RT], sm_l[NW][RT];
    __shared__ int sm_last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int head = blockIdx.y;
    uint8_t* stage = smem + warp * STAGE;
    uint64_t* bar_k = &bars[0][warp];
    uint64_t* bar_v = &bars[1][warp];
    if (lane == 0) {
        mbar_init(bar_k, 1);
        mbar_init(bar_v, 1);
        fence_mbar_init();
    }
    __syncwarp();
    pdl_wait();

    const RowsItem it = p.items[blockIdx.x];
    const int start = it.start;
    const int n_full = it.kv_len / PT;      // blocks past this one are the open page

    auto issue = [&](int page, int j) {    // one lane: K (j = 0) or V half of a page
        uint64_t* bar = j ? bar_v : bar_k;
        const int64_t ph = int64_t(page) * p.kv_heads + head;
        mbar_arrive_expect_tx(bar, TX_HALF);
        tma_load_2d(stage + j * 8192, &tm, 0, int((ph * 2 + j) * PT), bar);
        bulk_g2s(stage + SC + j * 512, p.scales + (ph * 4 + 2 * j) * D, 512, bar);
    };
    int blk = it.blk0 + warp;
    if (lane == 0 && blk < it.blk1 && blk < n_full) {
        const int page = warp == 0 ? it.page[0] : warp == 1 ? it.page[1] : warp == 2 ? it.page[2] : it.page[3];
        issue(page, 0);
        issue(page, 1);
    }

    // Rows of this lane's columns: their positions (-1: no row) and the key range they see.
    int row_pos[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        int r = HL ? (2 * t + (c & 1)) & 3 : (c >> 1) * 8 + 2 * t + (c & 1);
        row_pos[c] = r < it.nrows ? start + (it.row0 + r) / p.gq : -1;
    }
    // B fragments of Q: column g of tile n, channels 32t .. 32t+31 in order.
    uint32_t qf[NT][16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = HL ? (g & 3) : n * 8 + g;
        if (r < it.nrows) {
            const int row = it.row0 + r, tok = row / p.gq;
            const __half* qp = p.q + int64_t(it.q_start + tok) * p.q_t + int64_t(head * p.gq + row - tok * p.gq) * p.q_h + 32 * t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(qp + 8 * i);
                qf[n][4 * i] = v.x; qf[n][4 * i + 1] = v.y; qf[n][4 * i + 2] = v.z; qf[n][4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) qf[n][i] = 0u;
        }
    }

    float acc[NT][8][4], m[NC], l[NC], alpha[NC];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[n][j][c] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.f;
    }
    auto score = [&](float v, int pos, int c) {
        const bool ok = pos <= row_pos[c] && (p.window == 0 || pos > row_pos[c] - p.window);
        return ok ? v * p.scale_log2 : -INFINITY;
    };
    auto rescale = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[n][j][c] *= alpha[2 * n + (c & 1)];
    };

    uint32_t phase = 0;
    bool ok = true;
    for (; ok && blk < it.blk1 && blk < n_full; blk += NW) {
        const bool more = blk + NW < it.blk1 && blk + NW < n_full;
        const int page = more && lane == 0 ? p.pages[it.page_off + blk + NW] : 0;   // read before it is needed
        if (!(ok = mbar_wait(bar_k, phase, p.err, 1))) {   // give up, but not while this page's V may still land
            mbar_wait(bar_v, phase, p.err, 1);
            mbar_wait(bar_k, phase, p.err, 1);
            break;
        }
        float x[NC][8];
        {
            uint32_t st[16], mn[16];       // steps and minima of channels 32t .. 32t+31
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 a = lds128(stage + SC + 256 + 64 * t + 16 * i), b = lds128(stage + SC + 64 * t + 16 * i);
                st[4 * i] = a.x; st[4 * i + 1] = a.y; st[4 * i + 2] = a.z; st[4 * i + 3] = a.w;
                mn[4 * i] = b.x; mn[4 * i + 1] = b.y; mn[4 * i + 2] = b.z; mn[4 * i + 3] = b.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r0 = 16 * i + g;
                const uint4 k0a = lds128(stage + r0 * 128 + (((2 * t) ^ g) << 4));
                const uint4 k0b = lds128(stage + r0 * 128 + (((2 * t + 1) ^ g) << 4));
                const uint4 k1a = lds128(stage + (r0 + 8) * 128 + (((2 * t) ^ g) << 4));
                const uint4 k1b = lds128(stage + (r0 + 8) * 128 + (((2 * t + 1) ^ g) << 4));
                const uint32_t w0[8] = {k0a.x, k0a.y, k0a.z, k0a.w, k0b.x, k0b.y, k0b.z, k0b.w};
                const uint32_t w1[8] = {k1a.x, k1a.y, k1a.z, k1a.w, k1b.x, k1b.y, k1b.z, k1b.w};
                float c[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t a0 = hfma2(u8x2_lo_to_f16x2(w0[k]), st[2 * k], mn[2 * k]);
                    const uint32_t a2 = hfma2(u8x2_hi_to_f16x2(w0[k]), st[2 * k + 1], mn[2 * k + 1]);
                    const uint32_t a1 = hfma2(u8x2_lo_to_f16x2(w1[k]), st[2 * k], mn[2 * k]);
                    const uint32_t a3 = hfma2(u8x2_hi_to_f16x2(w1[k]), st[2 * k + 1], mn[2 * k + 1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(c[n], a0, a1, a2, a3, qf[n][2 * k], qf[n][2 * k + 1]);
                }
                const int p0 = blk * PT + r0;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[2 * n + e][2 * i] = score(c[n][e], p0, 2 * n + e);
                        x[2 * n + e][2 * i + 1] = score(c[n][2 + e], p0 + 8, 2 * n + e);
                    }
            }
        }
        __syncwarp();
        if (more && lane == 0) {
            fence_proxy_async();
            issue(page, 0);
        }
        softmax_step<NC, 8>(x, m, l, alpha);
        rescale();
        if (!(ok = mbar_wait(bar_v, phase, p.err, 1))) {   // the K half just requested must land before exit
            if (more) mbar_wait(bar_k, phase ^ 1u, p.err, 1);
            break;
        }
        {
            const uint8_t* vs = stage + 8192;
            uint32_t sA[8], sB[8], mA[8], mB[8];   // channel 16g + 2j (A) and 16g + 2j + 1 (B), both halves
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 a = lds128(stage + SC + 768 + 32 * g + 16 * i), b = lds128(stage + SC + 512 + 32 * g + 16 * i);
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sA[4 * i + k] = __byte_perm(aw[k], 0, 0x1010);
                    sB[4 * i + k] = __byte_perm(aw[k], 0, 0x3232);
                    mA[4 * i + k] = __byte_perm(bw[k], 0, 0x1010);
                    mB[4 * i + k] = __byte_perm(bw[k], 0, 0x3232);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    b0[n] = movmatrix_trans(pack_p<HL>(x[2 * n][2 * i], x[2 * n + 1][2 * i], t));
                    b1[n] = movmatrix_trans(pack_p<HL>(x[2 * n][2 * i + 1], x[2 * n + 1][2 * i + 1], t));
                }
                const int ta = 16 * i + 2 * t;
                const uint4 vA = lds128(vs + ta * 128 + ((g ^ (ta & 7)) << 4));
                const uint4 vB = lds128(vs + (ta + 1) * 128 + ((g ^ ((ta + 1) & 7)) << 4));
                const uint4 vC = lds128(vs + (ta + 8) * 128 + ((g ^ (ta & 7)) << 4));
                const uint4 vD = lds128(vs + (ta + 9) * 128 + ((g ^ ((ta + 1) & 7)) << 4));
                const uint32_t wa[4] = {vA.x, vA.y, vA.z, vA.w}, wb[4] = {vB.x, vB.y, vB.z, vB.w};
                const uint32_t wc[4] = {vC.x, vC.y, vC.z, vC.w}, wd[4] = {vD.x, vD.y, vD.z, vD.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t ab[2] = {__byte_perm(wa[w], wb[w], 0x5140), __byte_perm(wa[w], wb[w], 0x7362)};
                    const uint32_t cd[2] = {__byte_perm(wc[w], wd[w], 0x5140), __byte_perm(wc[w], wd[w], 0x7362)};
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = 2 * w + e;
                        const uint32_t a0 = hfma2(u8x2_lo_to_f16x2(ab[e]), sA[j], mA[j]);
                        const uint32_t a1 = hfma2(u8x2_hi_to_f16x2(ab[e]), sB[j], mB[j]);
                        const uint32_t a2 = hfma2(u8x2_lo_to_f16x2(cd[e]), sA[j], mA[j]);
                        const uint32_t a3 = hfma2(u8x2_hi_to_f16x2(cd[e]), sB[j], mB[j]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16816(acc[n][j], a0, a1, a2, a3, b0[n], b1[n]);
                    }
                }
            }
        }
        __syncwarp();
        if (more && lane == 0) {
            fence_proxy_async();
            issue(page, 1);
        }
        phase ^= 1u;
    }
    // The open page, 16 fp16 tokens at a time (one tile per warp, the first to the warp whose turn it is), by the
    // item that holds its block.
    if (ok && it.blk1 > n_full && it.blk0 <= n_full) {
        const int tile = (warp - (n_full - it.blk0)) & (NW - 1), r0 = 16 * tile + g, base = n_full * PT;
        if (base + 16 * tile < it.kv_len) {
            const __half* tk = p.tails + half_off(it.tail, p.kv_heads, head, 0);
            const __half* tv = tk + HALF_ROW;
            const bool live0 = base + r0 < it.kv_len, live1 = base + r0 + 8 < it.kv_len;
            float x[NC][2];
            {
                uint32_t k0[16], k1[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
                    const uint4 a = live0 ? *reinterpret_cast<const uint4*>(tk + r0 * D + 32 * t + 8 * i) : z;
                    const uint4 b = live1 ? *reinterpret_cast<const uint4*>(tk + (r0 + 8) * D + 32 * t + 8 * i) : z;
                    k0[4 * i] = a.x; k0[4 * i + 1] = a.y; k0[4 * i + 2] = a.z; k0[4 * i + 3] = a.w;
                    k1[4 * i] = b.x; k1[4 * i + 1] = b.y; k1[4 * i + 2] = b.z; k1[4 * i + 3] = b.w;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_16816(c, k0[2 * k], k1[2 * k], k0[2 * k + 1], k1[2 * k + 1], qf[n][2 * k], qf[n][2 * k + 1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[2 * n + e][0] = score(c[e], base + r0, 2 * n + e);
                        x[2 * n + e][1] = score(c[2 + e], base + r0 + 8, 2 * n + e);
                    }
                }
            }
            softmax_step<NC, 2>(x, m, l, alpha);
            rescale();
            uint32_t v[4][8];
            const int ta = 16 * tile + 2 * t;
            const int tok[4] = {ta, ta + 1, ta + 8, ta + 9};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 z = make_uint4(0u, 0u, 0u, 0u);
                const bool in = base + tok[k] < it.kv_len;   // a slot that holds no token may hold anything
                const uint4 a = in ? *reinterpret_cast<const uint4*>(tv + tok[k] * D + 16 * g) : z;
                const uint4 b = in ? *reinterpret_cast<const uint4*>(tv + tok[k] * D + 16 * g + 8) : z;
                v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
                v[k][4] = b.x; v[k][5] = b.y; v[k][6] = b.z; v[k][7] = b.w;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t b0 = movmatrix_trans(pack_p<HL>(x[2 * n][0], x[2 * n + 1][0], t));
                const uint32_t b1 = movmatrix_trans(pack_p<HL>(x[2 * n][1], x[2 * n + 1][1], t));
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    mma_16816(acc[n][j], __byte_perm(v[0][j], v[1][j], 0x5410), __byte_perm(v[0][j], v[1][j], 0x7632),
                              __byte_perm(v[2][j], v[3][j], 0x5410), __byte_perm(v[2][j], v[3][j], 0x7632), b0, b1);
            }
        }
    }

    // ---- join the four warps
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 4);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 8);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 16);
    }
    if (HL) {   // low parts (lanes t >= 2) onto the high ones
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[0][j][c] += __shfl_xor_sync(0xffffffffu, acc[0][j][c], 2);
    }
    __syncthreads();                        // every stage is idle
    float* obuf = reinterpret_cast<float*>(smem);   // [NW][RT][D]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + 2 * t + e;
            if (r >= RT) continue;
            if (g == 0) {
                sm_m[warp][r] = m[2 * n + e];
                sm_l[warp][r] = l[2 * n + e];
            }
            float* o = obuf + (warp * RT + r) * D + 16 * g;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<float2*>(o + 2 * j) = make_float2(acc[n][j][e], acc[n][j][2 + e]);
        }
    __syncthreads();
    const int d0 = lane * 4;
    auto finish = [&](int r, float M, float L, float4 o) {   // one row, a warp: out and lse
        const int row = it.row0 + r, tok = row / p.gq, qh = head * p.gq + row - tok * p.gq;
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        const uint2 h = make_uint2(pack_f16x2(o.x * inv, o.y * inv), pack_f16x2(o.z * inv, o.w * inv));
        *reinterpret_cast<uint2*>(p.out + int64_t(it.q_start + tok) * p.o_t + int64_t(qh) * p.o_h + d0) = h;
        if (p.lse && lane == 0)
            p.lse[int64_t(it.q_start + tok) * p.q_heads + qh] =
                L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    };
    const int64_t slot = (int64_t(it.part0) * p.kv_heads + head * int64_t(it.n_splits));
    float* part = p.part + (slot + it.split) * p.tile_rows * PART;   // [part0 ..][head][split][row][PART]
    for (int r = warp; r < it.nrows; r += NW) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_m[w][r]);
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float wt = M == -INFINITY ? 0.f : exp2f(sm_m[w][r] - M);
            const float4 a = *reinterpret_cast<const float4*>(obuf + (w * RT + r) * D + d0);
            L += wt * sm_l[w][r];
            o.x += wt * a.x; o.y += wt * a.y; o.z += wt * a.z; o.w += wt * a.w;
        }
        if (it.n_splits == 1) {
            finish(r, M, L, o);
        } else {
            if (lane == 0) *reinterpret_cast<float2*>(part + r * PART) = make_float2(M, L);
            *reinterpret_cast<float4*>(part + r * PART + 4 + d0) = o;
        }
    }
    if (it.n_splits == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned* ctr = p.counters + int64_t(it.part0) * p.kv_heads + head;
        const unsigned prev = atomicAdd(ctr, 1u);
        sm_last = prev == unsigned(it.n_splits - 1);
        if (sm_last) *ctr = 0u;            // every split has arrived: ready for the next launch
    }
    __syncthreads();
    if (!sm_last) return;
    __threadfence();
    const float* all = p.part + slot * p.tile_rows * PART;
    const int64_t step = int64_t(p.tile_rows) * PART;
    for (int r = warp; r < it.nrows; r += NW) {
        const float* pr = all + r * PART;
        float M = -INFINITY;
        for (int k = lane; k < it.n_splits; k += 32) M = fmaxf(M, __ldcg(pr + k * step));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < it.n_splits; ++k) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + k * step));
            const float4 a = __ldcg(reinterpret_cast<const float4*>(pr + k * step + 4 + d0));
            const float wt = M == -INFINITY ? 0.f : exp2f(ml.x - M);
            L += wt * ml.y;
            o.x += wt * a.x; o.y += wt * a.y; o.z += wt * a.z; o.w += wt * a.w;
        }
        finish(r, M, L, o);
    }
}

}  // namespace rows
}  // namespace paged
}  // namespace nova

using namespace nova;
using namespace nova::paged;

namespace {

typedef void (*RowsKernel)(const rows::Params, const CUtensorMap);

int launch_rows(const rows::Params& p, const CUtensorMap& tm, const nova_paged_rows& s, cudaStream_t stream) {
    static const RowsKernel kernels[3] = {rows::paged_attn_rows_kernel<1, true>, rows::paged_attn_rows_kernel<1, false>,
                                          rows::paged_attn_rows_kernel<2, false>};
    static bool ready[kMaxDevices][3];     // shared-memory limit raised on this device
    const int which = s.rows_per_tile == 4 ? 0 : s.rows_per_tile == 8 ? 1 : 2;
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices || !ready[dev][which]) {
        if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kernels[which]), cudaFuncAttributeMaxDynamicSharedMemorySize, rows::SMEM) !=
            cudaSuccess)
            return check_launch("paged attention");
        if (dev >= 0 && dev < kMaxDevices) ready[dev][which] = true;
    }
    launch(kernels[which], dim3(unsigned(s.n), unsigned(p.kv_heads)), dim3(rows::THREADS), rows::SMEM, stream, p, tm);
    return check_launch("paged attention");
}

}  // namespace

extern "C" int nova_paged_attention(const nova_paged_attn_args* a, const nova_paged_plan_info* info, void* stream) {
    if (!a) return fail(NOVA_ERR_INVALID, "paged attention: args must not be NULL");
    if (int rc = check_cache("paged attention", a->codes, a->scales, a->tails, a->num_pages, a->num_tails, a->plan, info))
        return rc;
    if (a->sched < 0 || a->sched >= info->n_windows)
        return fail(NOVA_ERR_INVALID, "paged attention: the plan has %lld windows, asked for number %lld",
                    (long long)info->n_windows, (long long)a->sched);
    if (!info->tokens) return NOVA_OK;
    if (!a->q || !a->out) return fail(NOVA_ERR_INVALID, "paged attention: NULL q or out");
    if (!(a->scale > 0) || !(a->scale < 1e6)) return fail(NOVA_ERR_INVALID, "paged attention: scale must be positive");
    auto off = [](const void* p, int64_t al) { return reinterpret_cast<uintptr_t>(p) % al != 0; };
    if (off(a->q, 16) || off(a->out, 16) || off(a->lse, 4) || off(a->workspace, 16) || a->q_t_stride % 8 ||
        a->q_h_stride % 8 || a->o_t_stride % 8 || a->o_h_stride % 8)
        return fail(NOVA_ERR_ALIGN, "paged attention: pointers need 16-byte alignment, strides multiples of 8");
    // out: one place for each row, or rows of different CTAs would write over one another
    const int64_t t = a->o_t_stride, h = a->o_h_stride;
    const bool many_t = info->tokens > 1, many_h = info->q_heads > 1;
    if ((many_t && t < D) || (many_h && h < D) ||
        (many_t && many_h && (t < h ? h < t * (info->tokens - 1) + D : t < h * (info->q_heads - 1) + D)))
        return fail(NOVA_ERR_INVALID, "paged attention: rows of out overlap (strides %lld and %lld)", (long long)t, (long long)h);
    if (a->workspace_bytes < info->workspace_bytes || !a->workspace)
        return fail(NOVA_ERR_INVALID, "paged attention: workspace of %lld bytes, %lld are needed",
                    (long long)a->workspace_bytes, (long long)info->workspace_bytes);
    const int64_t code_rows = a->num_pages * info->kv_heads * 2 * PT;
    if (code_rows >= (1ll << 31))
        return fail(NOVA_ERR_UNSUPPORTED, "paged attention: %lld pages of %lld heads exceed 2^31 code rows",
                    (long long)a->num_pages, (long long)info->kv_heads);
    const nova_paged_schedule& s = info->sched[a->sched];
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (s.n_ctas)
        if (int rc = launch_tiles(a, info, s, st)) return rc;
    if (!s.rows[0].n && !s.rows[1].n) return NOVA_OK;
    rows::Params p{};
    p.q = static_cast<const __half*>(a->q);
    p.q_t = a->q_t_stride;
    p.q_h = a->q_h_stride;
    p.scales = static_cast<const __half*>(a->scales);
    p.tails = static_cast<const __half*>(a->tails);
    p.out = static_cast<__half*>(a->out);
    p.o_t = a->o_t_stride;
    p.o_h = a->o_h_stride;
    p.lse = static_cast<float*>(a->lse);
    p.pages = a->plan + info->page_off;
    p.q_heads = int(info->q_heads);
    p.kv_heads = int(info->kv_heads);
    p.gq = p.q_heads / p.kv_heads;
    p.window = int(s.window);
    p.scale_log2 = float(a->scale * 1.4426950408889634);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.err = reinterpret_cast<int*>(ws);
    CUtensorMap tm{};
    if (a->num_pages > 0)
        if (int rc = make_tmap_u8_rows128(&tm, a->codes, uint64_t(code_rows), PT)) return rc;
    for (const nova_paged_rows& list : s.rows) {
        p.items = reinterpret_cast<const RowsItem*>(a->plan + list.off);
        p.tile_rows = int(list.rows_per_tile);
        p.counters = reinterpret_cast<unsigned*>(ws + list.counters_off);
        p.part = reinterpret_cast<float*>(ws + list.parts_off);
        if (list.n)
            if (int rc = launch_rows(p, tm, list, st)) return rc;
    }
    return NOVA_OK;
}

extern "C" int nova_paged_attention_read_error(void* workspace, int* host_value) {
    if (!workspace || !host_value) return fail(NOVA_ERR_INVALID, "paged attention: NULL workspace or value");
    if (cudaMemcpy(host_value, workspace, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess ||
        cudaMemset(workspace, 0, sizeof(int)) != cudaSuccess)
        return check_launch("paged attention error word");
    return NOVA_OK;
}
