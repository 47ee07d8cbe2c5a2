// Controls of each request on its next-token logits (penalties for repeated
// tokens, token biases, grammar masks), and the history they read.
//
// One pass: a thread takes two vectors of 8 consecutive tokens of a row -- 16
// bytes of fp16 logits, 16 of history, 8 mask bits each -- and writes them once.
// Few tokens are in a history or biased, so a vector passes as it came with the
// mask applied to its words, and those tokens are then done one by one in fp32
// with one rounding (all tokens through fp32: 44 instructions each and 20.1 us
// for 64 rows of 151936 fp16 logits; this way 18.4; 16.4 since the biases are on
// their way while the vectors are written, 16.6 since the penalty divides; fewer
// registers a thread for more CTAs per SM are slower).  Bound by instruction issue and the latency of a few waves
// of CTAs, then HBM: 58.8 MB at 3.5 TB/s; one row is a launch and two
// dependent loads, 5.1 us.  Vectors start at the 16-byte boundary at or before
// the row (the row's first and last vector go token by token); a row whose
// logits, history and output do not share such a boundary goes token by token
// throughout.
#include "common.cuh"

namespace nova {
namespace logits {

constexpr int THREADS = 128;
constexpr int VEC = 8;                  // tokens per vector
constexpr int NV = 2;                   // vectors per thread: what a row costs besides its tokens is half as much
constexpr int CHUNK = THREADS * VEC * NV;   // tokens per CTA, and per bias list
static_assert(CHUNK == NOVA_LOGITS_CHUNK, "callers build the bias lists by this number");

struct Params {
    const uint8_t* logits;
    int64_t lstride;
    uint8_t* out;
    int64_t ostride;
    const int16_t* history;
    int64_t hstride;
    const float* repetition;
    const float* frequency;
    const float* presence;
    const int* bias_off;
    const int* bias_token;
    const float* bias_value;
    const uint32_t* allowed;
    int64_t n_masks, mask_stride;
    const int* allowed_row;
    int vocab, chunks;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

template <typename T>
struct alignas(16) Vec {
    T v[VEC];
};

template <typename T>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(const Params p) {
    __shared__ float bias_s[CHUNK];              // of the tokens whose bit is set
    __shared__ __align__(8) uint32_t biased_s[CHUNK / 32];
    const int row = blockIdx.y, chunk = blockIdx.x;
    const T* src = reinterpret_cast<const T*>(p.logits) + row * p.lstride;
    T* dst = reinterpret_cast<T*>(p.out) + row * p.ostride;
    const int16_t* hist = p.history ? p.history + row * p.hstride : nullptr;
    // Tokens before the row that its first vector would cover, and whether every pointer agrees on it.
    const int lead = int(hist ? reinterpret_cast<uintptr_t>(hist) / 2 % VEC : reinterpret_cast<uintptr_t>(src) / sizeof(T) % VEC);
    const bool vec = (reinterpret_cast<uintptr_t>(src) - lead * sizeof(T)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(dst) - lead * sizeof(T)) % 16 == 0;
    const int base = chunk * CHUNK - lead;                     // first token of this CTA
    if (base >= p.vocab) return;
    auto first = [&](int q) { return base + (q * THREADS + int(threadIdx.x)) * VEC; };   // of vector q
    auto whole = [&](int q) { return vec && first(q) >= 0 && first(q) + VEC <= p.vocab; };
    pdl_wait();

    // loads that nothing waits for, all in flight
    Vec<T> x[NV];
    uint4 h[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        h[q] = make_uint4(0u, 0u, 0u, 0u);
        if (!whole(q)) continue;
        const uint4* s = reinterpret_cast<const uint4*>(src + first(q));
#pragma unroll
        for (int i = 0; i < int(sizeof(x[q]) / 16); ++i) reinterpret_cast<uint4*>(&x[q])[i] = s[i];
        if (hist) h[q] = *reinterpret_cast<const uint4*>(hist + first(q));
    }
    const int which = !p.allowed ? -1 : p.allowed_row ? p.allowed_row[row] : row;
    // mask words of each vector's tokens (no mask: all set; none allowed: none set)
    uint32_t mask[NV][2];
    auto shift = [&](int q) { return max(first(q), 0) & 31; };
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        mask[q][0] = mask[q][1] = which < p.n_masks ? ~0u : 0u;
        if (which < 0 || which >= p.n_masks) continue;
        const uint32_t* m = p.allowed + which * p.mask_stride;
        const int w = max(first(q), 0) >> 5, words = (p.vocab + 31) / 32;
        mask[q][0] = w < words ? m[w] : 0u;
        mask[q][1] = shift(q) > 32 - VEC && w + 1 < words ? m[w + 1] : 0u;
    }
    const float rep = p.repetition ? p.repetition[row] : 1.f;
    const float freq = p.frequency ? p.frequency[row] : 0.f;
    const float pres = p.presence ? p.presence[row] : 0.f;
    // Biases of this CTA's tokens: they lie in its list and, with a lead, in the one before.  Each thread's first is
    // on its way while the vectors are written.
    int e = 0, e1 = 0, at = -1;
    float value = 0.f;
    if (p.bias_off) {
        const int* off = p.bias_off + int64_t(row) * p.chunks;
        e = off[min(max(chunk - (lead > 0), 0), p.chunks)] + int(threadIdx.x);
        e1 = off[min(chunk + 1, p.chunks)];
        if (threadIdx.x < CHUNK / 32) biased_s[threadIdx.x] = 0u;
        __syncthreads();
        if (e < e1) {
            value = p.bias_value[e];
            at = p.bias_token[e] - base;
        }
    }
    // Most tokens are neither in the history nor biased: they leave as they came, unconverted, in whole vectors.
    uint32_t keep = 0u, todo = 0u;                             // 8 bits per vector: the mask's; tokens that change
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int t0 = first(q);
        const uint32_t k8 = __funnelshift_r(mask[q][0], mask[q][1], shift(q)) << (max(t0, 0) - t0) & 0xFFu;
        if (whole(q)) {
            const uint32_t hw[4] = {h[q].x, h[q].y, h[q].z, h[q].w};
            if (hw[0] | hw[1] | hw[2] | hw[3]) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    todo |= (hw[i] & 0xFFFFu ? 1u << (VEC * q + 2 * i) : 0u) | (hw[i] >> 16 ? 2u << (VEC * q + 2 * i) : 0u);
            }
            if (k8 != 0xFFu) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&x[q]);
                auto ones = [&](int i) { return uint32_t(int(k8 << (31 - i)) >> 31); };   // all bits of token i's mask bit
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int k = 0; k < VEC / 2; ++k) {
                        const uint32_t m = __byte_perm(ones(2 * k), ones(2 * k + 1), 0x5410);
                        w[k] = (w[k] & m) | (0xFC00FC00u & ~m);        // fp16 -inf
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) w[i] = (w[i] & ones(i)) | (0xFF800000u & ~ones(i));
                }
            }
            uint4* d = reinterpret_cast<uint4*>(dst + t0);
#pragma unroll
            for (int i = 0; i < int(sizeof(x[q]) / 16); ++i) d[i] = reinterpret_cast<const uint4*>(&x[q])[i];
            keep |= k8 << VEC * q;
        } else {              // token by token, those of the row
            const uint32_t in = t0 >= p.vocab || t0 + VEC <= 0
                                    ? 0u
                                    : (0xFFu << max(-t0, 0) & 0xFFu) & (0xFFu >> max(t0 + VEC - p.vocab, 0));
            for (uint32_t no = in & ~k8; no; no &= no - 1) dst[t0 + __ffs(no) - 1] = from_float<T>(-INFINITY);
            todo |= (in & k8) << VEC * q;
            keep |= (in & k8) << VEC * q;
        }
    }
    uint32_t biased = 0u;
    if (p.bias_off) {
        while (e < e1) {
            if (at >= 0 && at < CHUNK) {
                bias_s[at] = value;
                atomicOr(&biased_s[at / 32], 1u << (at % 32));     // set bits do not depend on the order
            }
            e += THREADS;
            if (e < e1) {
                value = p.bias_value[e];
                at = p.bias_token[e] - base;
            }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NV; ++q)
            biased |= uint32_t(reinterpret_cast<const uint8_t*>(biased_s)[q * THREADS + threadIdx.x]) << VEC * q;
    }
    // The others follow one by one, read again (an output that is the input still holds them).
    todo = (todo | biased) & keep;
    if (!todo) return;
    for (; todo; todo &= todo - 1) {
        const int i = __ffs(todo) - 1, own = (i / VEC * THREADS + int(threadIdx.x)) * VEC + i % VEC, t = base + own;
        float v = to_float<T>(src[t]);
        const int seen = hist ? hist[t] : 0, times = seen & 0x7FFF;
        if (seen) v = v > 0.f ? div_rn(v, rep) : v * rep;
        v -= times ? fmaf(freq, float(times), pres) : 0.f;
        if (biased >> i & 1u) v += bias_s[own];
        dst[t] = from_float<T>(v);
    }
}

// A count or a prompt bit lives in half of a 32-bit word; both updates are
// whole-number atomics on that word, so their order does not matter.  The
// offsets are device data that the host has not seen: what they name outside the
// n_tokens tokens is not read.
__global__ void history_add_kernel(int16_t* history, int64_t stride, const int64_t* tokens, int64_t n_tokens,
                                   const int* off, int vocab, int prompt) {
    pdl_wait();
    const int row = blockIdx.y;
    const int64_t first = off ? max(off[row], 0) : row, end = off ? min(int64_t(off[row + 1]), n_tokens) : row + 1;
    for (int64_t i = first + blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < end; i += int64_t(gridDim.x) * blockDim.x) {
        const int64_t t = tokens[i];
        if (t < 0 || t >= vocab) continue;
        const uintptr_t at = reinterpret_cast<uintptr_t>(history + row * stride + t);
        unsigned* word = reinterpret_cast<unsigned*>(at & ~uintptr_t(3));
        const int shift = int(at & 2) * 8;
        if (prompt) {
            atomicOr(word, 0x8000u << shift);
            continue;
        }
        unsigned was = *reinterpret_cast<volatile unsigned*>(word);
        for (;;) {   // every failed exchange is another thread's success, so this ends
            if (((was >> shift) & 0x7FFFu) == 0x7FFFu) break;
            const unsigned got = atomicCAS(word, was, was + (1u << shift));
            if (got == was) break;
            was = got;
        }
    }
}

}  // namespace logits
}  // namespace nova

using namespace nova;

extern "C" int nova_adjust_logits(const nova_logits_args* a, void* stream) {
    using namespace nova::logits;
    if (!a) return fail(NOVA_ERR_INVALID, "adjust logits: args must not be NULL");
    if (a->rows < 0 || a->vocab < 1 || a->vocab >= (1ll << 31) - CHUNK || a->rows > 65535)
        return fail(NOVA_ERR_INVALID, "adjust logits: rows=%lld, vocab=%lld", (long long)a->rows, (long long)a->vocab);
    if (!a->rows) return NOVA_OK;
    if (!a->logits || !a->out) return fail(NOVA_ERR_INVALID, "adjust logits: NULL logits or out");
    if (a->rows > 1 && (a->logits_stride < a->vocab || a->out_stride < a->vocab || (a->history && a->history_stride < a->vocab)))
        return fail(NOVA_ERR_INVALID, "adjust logits: row strides below the vocabulary");
    if (a->allowed && (a->n_masks < 1 || a->mask_stride < (a->vocab + 31) / 32))
        return fail(NOVA_ERR_INVALID, "adjust logits: masks of %lld words, %lld are needed", (long long)a->mask_stride,
                    (long long)((a->vocab + 31) / 32));
    if (a->bias_off && (!a->bias_token || !a->bias_value))
        return fail(NOVA_ERR_INVALID, "adjust logits: NULL bias tokens or values");
    auto off = [](const void* p, int64_t al) { return reinterpret_cast<uintptr_t>(p) % al != 0; };
    const int64_t el = a->logits_fp32 ? 4 : 2;
    if (off(a->logits, el) || off(a->out, el) || off(a->history, 2) || off(a->allowed, 4))
        return fail(NOVA_ERR_ALIGN, "adjust logits: pointers need the alignment of their elements");
    Params p{};
    p.logits = static_cast<const uint8_t*>(a->logits);
    p.lstride = a->logits_stride;
    p.out = static_cast<uint8_t*>(a->out);
    p.ostride = a->out_stride;
    p.history = static_cast<const int16_t*>(a->history);
    p.hstride = a->history_stride;
    p.repetition = static_cast<const float*>(a->repetition);
    p.frequency = static_cast<const float*>(a->frequency);
    p.presence = static_cast<const float*>(a->presence);
    p.bias_off = a->bias_off;
    p.bias_token = a->bias_token;
    p.bias_value = static_cast<const float*>(a->bias_value);
    p.allowed = static_cast<const uint32_t*>(a->allowed);
    p.n_masks = a->n_masks;
    p.mask_stride = a->mask_stride;
    p.allowed_row = a->allowed_row;
    p.vocab = int(a->vocab);
    p.chunks = int((a->vocab + CHUNK - 1) / CHUNK);
    const dim3 grid(unsigned((a->vocab + VEC - 1 + CHUNK - 1) / CHUNK), unsigned(a->rows));
    launch(a->logits_fp32 ? adjust_logits_kernel<float> : adjust_logits_kernel<__half>, grid, dim3(THREADS), 0,
           static_cast<cudaStream_t>(stream), p);
    return check_launch("adjust logits");
}

extern "C" int nova_history_add(void* history, int64_t history_stride, const int64_t* tokens, const int32_t* off,
                                int64_t n_tokens, int64_t rows, int64_t vocab, int prompt, void* stream) {
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab >= (1ll << 31) || n_tokens < 0)
        return fail(NOVA_ERR_INVALID, "history add: rows=%lld, vocab=%lld, tokens=%lld", (long long)rows,
                    (long long)vocab, (long long)n_tokens);
    if (!rows || !n_tokens) return NOVA_OK;
    if (!history || !tokens) return fail(NOVA_ERR_INVALID, "history add: NULL history or tokens");
    if (rows > 1 && history_stride < vocab) return fail(NOVA_ERR_INVALID, "history add: row stride below the vocabulary");
    if (!off && n_tokens != rows) return fail(NOVA_ERR_INVALID, "history add: one token per row without offsets");
    if (reinterpret_cast<uintptr_t>(history) % 2 || reinterpret_cast<uintptr_t>(tokens) % 8 ||
        reinterpret_cast<uintptr_t>(off) % 4)
        return fail(NOVA_ERR_ALIGN, "history add: pointers need the alignment of their elements");
    const int64_t per_row = off ? (n_tokens + rows - 1) / rows : 1;
    const unsigned gx = unsigned(std::min<int64_t>(32, (per_row + 255) / 256));
    launch(logits::history_add_kernel, dim3(gx, unsigned(rows)), dim3(off ? 256 : 32), 0,
           static_cast<cudaStream_t>(stream), static_cast<int16_t*>(history), history_stride, tokens, n_tokens,
           static_cast<const int*>(off), int(vocab), prompt);
    return check_launch("history add");
}
