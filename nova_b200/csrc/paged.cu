// Paged int8 cache: q|k|v rows of a step's new tokens into it (per-head norm,
// RoPE, quantization of the pages that fill), and stored values back out.
//
// Both kernels move each byte once and compute little, so what bounds them is
// HBM for prompts and the latency of a launch and two dependent loads for
// single tokens.  One thread holds channels 4c..4c+3 and 64+4c..64+4c+3 of a
// row (c = lane % 16): the two halves that RoPE combines are then in one
// thread, a row is two 128-byte requests of a half warp, and the mean of
// squares is four shuffles.  Measured: 8 prompts of 130 to 1021 tokens at 48
// heads append in 31 us (issue slots 69 % busy; 63 MB of DRAM traffic) and read
// back in 8.6; together 123 MB at 3.1 TB/s.  One token of each of 64 requests:
// 5 us each, of which a launch is 2 to 3.
#include "paged.cuh"

namespace nova {
namespace paged {

constexpr int THREADS = 256;
constexpr int RH = 4;           // heads of one token that a half warp takes
constexpr int ITEMS = 16;       // such items per CTA of the row part

struct AppendParams {
    const __half* qkv;
    int64_t qkv_stride;
    const __half* wq;
    const __half* wk;
    float eps;
    const __half* cos;
    const __half* sin;
    __half* q;
    int64_t q_stride;
    uint8_t* codes;
    __half* scales;
    __half* tails;
    const int* pos;
    const OpenToken* open;
    const Block* blocks;
    int tokens, n_open, n_write, q_heads, kv_heads;
    int row_ctas;
};

struct Row8 {                   // channels 4c..4c+3 and 64+4c..64+4c+3 of one row
    uint2 lo, hi;
};

__device__ __forceinline__ Row8 load_row(const __half* p, int c) {
    Row8 r;
    r.lo = *reinterpret_cast<const uint2*>(p + 4 * c);
    r.hi = *reinterpret_cast<const uint2*>(p + 64 + 4 * c);
    return r;
}
__device__ __forceinline__ void store_row(__half* p, int c, const Row8& r) {
    *reinterpret_cast<uint2*>(p + 4 * c) = r.lo;
    *reinterpret_cast<uint2*>(p + 64 + 4 * c) = r.hi;
}
__device__ __forceinline__ void unpack(const Row8& r, float (&x)[8]) {
    const uint32_t w[4] = {r.lo.x, r.lo.y, r.hi.x, r.hi.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ Row8 pack(const float (&x)[8]) {
    Row8 r;
    r.lo = make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
    r.hi = make_uint2(pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
    return r;
}

// RMSNorm (norm; w: the weights) and RoPE (rope) of one row held by a half warp,
// in fp32 and rounded to fp16 once: the reference rounds after the norm, after
// the weight and after each rotation product, which costs half a unit in the
// last place each time and nothing here needs its bits.
__device__ __forceinline__ Row8 norm_rope_row(const Row8& in, bool norm, const float (&w)[8], bool rope,
                                              const float (&cs)[8], const float (&sn)[8], float eps) {
    float x[8];
    unpack(in, x);
    float ss = 0.f;              // summed whether it is used or not: the other half warp may want its norm
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (norm) {
        const float r = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
    }
    if (rope) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = x[i] * cs[i] - x[i + 4] * sn[i];
            y[i + 4] = x[i + 4] * cs[i + 4] + x[i] * sn[i + 4];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i];
    }
    return pack(x);
}

// Code of a finite value: rint((v - low) / step) of the framework's quantizer, bit
// for bit.  The quotient by the reciprocal is within 4e-5 of the divided one (it is
// at most 255), so only one that close to a tie is divided; adding 1.5 * 2^23
// rounds to the nearest even integer and leaves it in the low mantissa bits.
__device__ __forceinline__ uint32_t code_of(float v, float low, float step, float inv) {
    constexpr float MAGIC = 12582912.0f;
    const float d = v - low, q = d * inv;
    float t = __fadd_rn(q, MAGIC);
    if (fabsf(q - __fadd_rn(t, -MAGIC)) > 0.4999f) t = __fadd_rn(div_rn(d, step), MAGIC);
    return __float_as_uint(t) & 0xFFu;
}

// A NaN among a channel's tokens is its minimum and maximum: the page's scale says
// so, and no code stands for a number that was none.
__device__ __forceinline__ uint32_t hmin2u(uint32_t a, uint32_t b) {
    __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmax2u(uint32_t a, uint32_t b) {
    __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}

// CTAs [0, row_ctas): 16 groups of 4 heads of a token each, one per half warp:
// query heads, then K and V heads (of tokens whose page stays open: into its tail
// buffer).  The others: K or V of one (block that the step completes, KV head),
// held in registers (4 tokens x 8 channels a thread); its minimum and maximum per
// channel go through shared memory once, and codes leave as 4-byte pieces of
// 128-byte rows.
__global__ void __launch_bounds__(THREADS, 4) paged_append_kernel(const AppendParams p) {
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 15, part = warp * 2 + (lane >> 4);
    const Row8 zero{make_uint2(0u, 0u), make_uint2(0u, 0u)};
    if (int(blockIdx.x) < p.row_ctas) {
        const int gq = (p.q_heads + RH - 1) / RH, gk = (p.kv_heads + RH - 1) / RH;
        const int nq = p.tokens * gq, n = nq + p.n_open * 2 * gk;
        const int at = int(blockIdx.x) * ITEMS + part;
        const bool live = at < n, query = at < nq;
        int tok = 0, h0 = 0, pos = 0, kind = 0, tail = 0;                     // kind: Q, K, V
        if (query) {
            tok = at / gq;
            h0 = (at - tok * gq) * RH;
            pos = p.cos ? p.pos[tok] : 0;
        } else if (live) {
            const int o = (at - nq) / (2 * gk), grp = (at - nq) - o * 2 * gk;
            const OpenToken t = p.open[o];
            kind = grp < gk ? 1 : 2;
            h0 = (grp < gk ? grp : grp - gk) * RH;
            tok = t.row;
            pos = t.pos;
            tail = t.tail;
        }
        const int heads = query ? p.q_heads : p.kv_heads;
        const __half* src = p.qkv + tok * p.qkv_stride + (h0 + (kind == 0 ? 0 : p.q_heads + (kind == 1 ? 0 : p.kv_heads))) * D;
        Row8 r[RH];
#pragma unroll
        for (int i = 0; i < RH; ++i) r[i] = live && h0 + i < heads ? load_row(src + i * D, c) : zero;
        const __half* wp = kind == 0 ? p.wq : kind == 1 ? p.wk : nullptr;
        const bool rope = p.cos && kind < 2;
        float w[8], cs[8], sn[8];
        unpack(wp ? load_row(wp, c) : zero, w);
        unpack(rope ? load_row(p.cos + int64_t(pos) * D, c) : zero, cs);
        unpack(rope ? load_row(p.sin + int64_t(pos) * D, c) : zero, sn);
#pragma unroll
        for (int i = 0; i < RH; ++i) {
            const Row8 y = norm_rope_row(r[i], wp, w, rope, cs, sn, p.eps);
            __half* dst = kind == 0 ? p.q + tok * p.q_stride + (h0 + i) * D
                                    : p.tails + half_off(tail, p.kv_heads, h0 + i, kind - 1) + pos % PT * D;
            if (live && h0 + i < heads) store_row(dst, c, y);
        }
        return;
    }
    const int item = (blockIdx.x - p.row_ctas) / (2 * p.kv_heads), hj = (blockIdx.x - p.row_ctas) % (2 * p.kv_heads);
    const int head = hj >> 1, j = hj & 1;
    const Block blk = p.blocks[item];
    const int b0 = blk.blk * PT;
    const __half* src = p.qkv + (p.q_heads + j * p.kv_heads + head) * int64_t(D) + int64_t(blk.row - blk.first) * p.qkv_stride;
    const __half* old = p.tails + half_off(blk.tail_in, p.kv_heads, head, j);
    Row8 r[4], cs[4], sn[4];
    bool fresh[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int slot = i * 16 + part, pos = b0 + slot;
        fresh[i] = pos >= blk.first;
        cs[i] = sn[i] = zero;
        if (fresh[i]) {
            r[i] = load_row(src + int64_t(pos) * p.qkv_stride, c);
            if (j == 0 && p.cos) {
                cs[i] = load_row(p.cos + int64_t(pos) * D, c);
                sn[i] = load_row(p.sin + int64_t(pos) * D, c);
            }
        } else {                                               // the open page's token
            r[i] = load_row(old + slot * D, c);
        }
    }
    if (j == 0) {
        float w[8], cf[8], sf[8];
        unpack(p.wk ? load_row(p.wk, c) : zero, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!__any_sync(0xffffffffu, fresh[i])) continue;
            unpack(cs[i], cf);
            unpack(sn[i], sf);
            const Row8 y = norm_rope_row(r[i], p.wk, w, p.cos, cf, sf, p.eps);
            if (fresh[i]) r[i] = y;
        }
    }
    __shared__ __align__(8) uint32_t lims[8][2][D / 2];   // per warp: minima, maxima of each channel pair
    uint32_t mn[4], mx[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t w[4] = {k < 2 ? (k ? r[0].lo.y : r[0].lo.x) : (k == 2 ? r[0].hi.x : r[0].hi.y),
                               k < 2 ? (k ? r[1].lo.y : r[1].lo.x) : (k == 2 ? r[1].hi.x : r[1].hi.y),
                               k < 2 ? (k ? r[2].lo.y : r[2].lo.x) : (k == 2 ? r[2].hi.x : r[2].hi.y),
                               k < 2 ? (k ? r[3].lo.y : r[3].lo.x) : (k == 2 ? r[3].hi.x : r[3].hi.y)};
        mn[k] = hmin2u(hmin2u(w[0], w[1]), hmin2u(w[2], w[3]));
        mx[k] = hmax2u(hmax2u(w[0], w[1]), hmax2u(w[2], w[3]));
        mn[k] = hmin2u(mn[k], __shfl_xor_sync(0xffffffffu, mn[k], 16));
        mx[k] = hmax2u(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 16));
    }
    if (lane < 16) {
        *reinterpret_cast<uint2*>(&lims[warp][0][2 * c]) = make_uint2(mn[0], mn[1]);
        *reinterpret_cast<uint2*>(&lims[warp][0][32 + 2 * c]) = make_uint2(mn[2], mn[3]);
        *reinterpret_cast<uint2*>(&lims[warp][1][2 * c]) = make_uint2(mx[0], mx[1]);
        *reinterpret_cast<uint2*>(&lims[warp][1][32 + 2 * c]) = make_uint2(mx[2], mx[3]);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const uint2 a = *reinterpret_cast<const uint2*>(&lims[w][0][2 * c]);
        const uint2 b = *reinterpret_cast<const uint2*>(&lims[w][0][32 + 2 * c]);
        const uint2 d = *reinterpret_cast<const uint2*>(&lims[w][1][2 * c]);
        const uint2 e = *reinterpret_cast<const uint2*>(&lims[w][1][32 + 2 * c]);
        mn[0] = hmin2u(mn[0], a.x); mn[1] = hmin2u(mn[1], a.y); mn[2] = hmin2u(mn[2], b.x); mn[3] = hmin2u(mn[3], b.y);
        mx[0] = hmax2u(mx[0], d.x); mx[1] = hmax2u(mx[1], d.y); mx[2] = hmax2u(mx[2], e.x); mx[3] = hmax2u(mx[3], e.y);
    }
    float low[8], step[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 a = __half22float2(*reinterpret_cast<__half2*>(&mn[k]));
        const float2 b = __half22float2(*reinterpret_cast<__half2*>(&mx[k]));
        low[2 * k] = a.x;
        low[2 * k + 1] = a.y;
        step[2 * k] = fmaxf(div_rn(b.x - a.x, 255.0f), 1e-8f);
        step[2 * k + 1] = fmaxf(div_rn(b.y - a.y, 255.0f), 1e-8f);
    }
    const int page = blk.page;
    float inv[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) inv[k] = div_rn(1.0f, step[k]);
    uint8_t* codes = p.codes + half_off(page, p.kv_heads, head, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x[8];
        unpack(r[i], x);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k >> 2] |= code_of(x[k], low[k], step[k], inv[k]) << (8 * (k & 3));
        uint8_t* row = codes + (i * 16 + part) * D;
        *reinterpret_cast<uint32_t*>(row + 4 * c) = w[0];
        *reinterpret_cast<uint32_t*>(row + 64 + 4 * c) = w[1];
    }
    if (part == 0) {
        __half* sc = p.scales + ((int64_t(page) * p.kv_heads + head) * 4 + 2 * j) * D;
        store_row(sc, c, Row8{make_uint2(mn[0], mn[1]), make_uint2(mn[2], mn[3])});
        store_row(sc + D, c, pack(step));
    }
}

// K or V of one (block, KV head) as fp16 rows.
__global__ void __launch_bounds__(THREADS)
    paged_read_kernel(const uint8_t* codes, const __half* scales, const __half* tails, const Block* blocks, int kv_heads,
                      __half* k_out, __half* v_out) {
    pdl_wait();
    const int lane = threadIdx.x & 31, c = lane & 15, part = (threadIdx.x >> 5) * 2 + (lane >> 4);
    const int item = blockIdx.x / (2 * kv_heads), hj = blockIdx.x % (2 * kv_heads), head = hj >> 1, j = hj & 1;
    const Block blk = blocks[item];
    const int b0 = blk.blk * PT, from = blk.first - b0;
    const int64_t stride = int64_t(kv_heads) * D;
    __half* out = (j ? v_out : k_out) + head * D + int64_t(blk.row - blk.first + b0) * stride;   // of the block's slot 0
    if (blk.page < 0) {
        const __half* src = tails + half_off(blk.tail_out, kv_heads, head, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int slot = i * 16 + part;
            if (slot >= from && b0 + slot < blk.kv_len) store_row(out + slot * stride, c, load_row(src + slot * D, c));
        }
        return;
    }
    const uint8_t* src = codes + half_off(blk.page, kv_heads, head, j);
    const __half* sc = scales + ((int64_t(blk.page) * kv_heads + head) * 4 + 2 * j) * D;
    const Row8 mn = load_row(sc, c), st = load_row(sc + D, c);
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = *reinterpret_cast<const uint32_t*>(src + (i * 16 + part) * D + 4 * c);
        b[i] = *reinterpret_cast<const uint32_t*>(src + (i * 16 + part) * D + 64 + 4 * c);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int slot = i * 16 + part;
        if (slot < from) continue;
        Row8 r;   // fp16(code * step + min), one rounding
        r.lo = make_uint2(hfma2(u8x2_lo_to_f16x2(a[i]), st.lo.x, mn.lo.x), hfma2(u8x2_hi_to_f16x2(a[i]), st.lo.y, mn.lo.y));
        r.hi = make_uint2(hfma2(u8x2_lo_to_f16x2(b[i]), st.hi.x, mn.hi.x), hfma2(u8x2_hi_to_f16x2(b[i]), st.hi.y, mn.hi.y));
        store_row(out + slot * stride, c, r);
    }
}

static bool misaligned(const void* p, int64_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// Cache pointers and sizes against what the plan uses.
int check_cache(const char* what, const void* codes, const void* scales, const void* tails, int64_t num_pages,
                int64_t num_tails, const void* plan, const nova_paged_plan_info* info) {
    if (!info || !plan) return fail(NOVA_ERR_INVALID, "%s: plan and info must not be NULL", what);
    if (info->kv_heads < 1 || info->q_heads < 1) return fail(NOVA_ERR_INVALID, "%s: info was not filled", what);
    if (info->max_page >= num_pages)
        return fail(NOVA_ERR_INVALID, "%s: the plan uses page %lld of %lld", what, (long long)info->max_page,
                    (long long)num_pages);
    if (info->max_tail >= num_tails)
        return fail(NOVA_ERR_INVALID, "%s: the plan uses tail buffer %lld of %lld", what, (long long)info->max_tail,
                    (long long)num_tails);
    if ((info->max_page >= 0 && (!codes || !scales)) || (info->max_tail >= 0 && !tails))
        return fail(NOVA_ERR_INVALID, "%s: NULL cache pointer", what);
    if (misaligned(codes, 16) || misaligned(scales, 16) || misaligned(tails, 16) || misaligned(plan, 16))
        return fail(NOVA_ERR_ALIGN, "%s: cache and plan need 16-byte alignment", what);
    return NOVA_OK;
}

}  // namespace paged
}  // namespace nova

using namespace nova;
using namespace nova::paged;

extern "C" int nova_paged_append(const nova_paged_append_args* a, const nova_paged_plan_info* info, void* stream) {
    if (!a) return fail(NOVA_ERR_INVALID, "paged append: args must not be NULL");
    if (int rc = check_cache("paged append", a->codes, a->scales, a->tails, a->num_pages, a->num_tails, a->plan, info))
        return rc;
    if (!info->tokens) return NOVA_OK;
    const int64_t width = (info->q_heads + 2 * info->kv_heads) * D;
    if (!a->qkv || !a->q_out) return fail(NOVA_ERR_INVALID, "paged append: NULL qkv or q_out");
    if (!a->cos != !a->sin) return fail(NOVA_ERR_INVALID, "paged append: cos and sin go together");
    if (a->cos && info->max_pos >= a->rope_len)
        return fail(NOVA_ERR_INVALID, "paged append: position %lld is past the rotation table's %lld rows",
                    (long long)info->max_pos, (long long)a->rope_len);
    if (a->qkv_stride < width || a->q_t_stride < info->q_heads * D)
        return fail(NOVA_ERR_INVALID, "paged append: row strides below the row length");
    if (misaligned(a->qkv, 16) || misaligned(a->q_out, 16) || a->qkv_stride % 8 || a->q_t_stride % 8 ||
        misaligned(a->q_norm_weight, 16) || misaligned(a->k_norm_weight, 16) || misaligned(a->cos, 16) ||
        misaligned(a->sin, 16))
        return fail(NOVA_ERR_ALIGN, "paged append: pointers need 16-byte alignment, strides multiples of 8");
    AppendParams p{};
    p.qkv = static_cast<const __half*>(a->qkv);
    p.qkv_stride = a->qkv_stride;
    p.wq = static_cast<const __half*>(a->q_norm_weight);
    p.wk = static_cast<const __half*>(a->k_norm_weight);
    p.eps = float(a->eps);
    p.cos = static_cast<const __half*>(a->cos);
    p.sin = static_cast<const __half*>(a->sin);
    p.q = static_cast<__half*>(a->q_out);
    p.q_stride = a->q_t_stride;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<__half*>(a->scales);
    p.tails = static_cast<__half*>(a->tails);
    p.pos = a->plan + info->pos_off;
    p.open = reinterpret_cast<const OpenToken*>(a->plan + info->open_off);
    p.n_open = int(info->n_open);
    p.blocks = reinterpret_cast<const Block*>(a->plan + info->write_off);
    p.tokens = int(info->tokens);
    p.n_write = int(info->n_write);
    p.q_heads = int(info->q_heads);
    p.kv_heads = int(info->kv_heads);
    const int64_t rows = info->tokens * ((info->q_heads + RH - 1) / RH) + info->n_open * 2 * ((info->kv_heads + RH - 1) / RH);
    const int64_t row_ctas = (rows + ITEMS - 1) / ITEMS;
    const int64_t grid = row_ctas + info->n_write * 2 * info->kv_heads;
    if (grid >= (1ll << 31)) return fail(NOVA_ERR_UNSUPPORTED, "paged append: too many tokens in one step");
    p.row_ctas = int(row_ctas);
    launch(paged_append_kernel, dim3(unsigned(grid)), dim3(THREADS), 0, static_cast<cudaStream_t>(stream), p);
    return check_launch("paged append");
}

extern "C" int nova_paged_read(const void* codes, const void* scales, const void* tails, int64_t num_pages,
                               int64_t num_tails, const int32_t* plan, const nova_paged_plan_info* info, void* k_out,
                               void* v_out, void* stream) {
    if (int rc = check_cache("paged read", codes, scales, tails, num_pages, num_tails, plan, info)) return rc;
    if (!info->n_read) return NOVA_OK;
    if (!k_out || !v_out) return fail(NOVA_ERR_INVALID, "paged read: NULL output");
    if (misaligned(k_out, 16) || misaligned(v_out, 16))
        return fail(NOVA_ERR_ALIGN, "paged read: outputs need 16-byte alignment");
    const int64_t grid = info->n_read * 2 * info->kv_heads;
    if (grid >= (1ll << 31)) return fail(NOVA_ERR_UNSUPPORTED, "paged read: too many rows in one call");
    launch(paged_read_kernel, dim3(unsigned(grid)), dim3(THREADS), 0, static_cast<cudaStream_t>(stream),
           static_cast<const uint8_t*>(codes), static_cast<const __half*>(scales), static_cast<const __half*>(tails),
           reinterpret_cast<const Block*>(plan + info->read_off), int(info->kv_heads), static_cast<__half*>(k_out),
           static_cast<__half*>(v_out));
    return check_launch("paged read");
}
