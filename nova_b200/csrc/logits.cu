// Controls of each request on its next-token logits (penalties for repeated
// tokens, token biases, grammar masks), and the history they read.
//
// One pass: a thread takes 8 consecutive tokens of a row -- 16 bytes of fp16
// logits, 16 of history, 8 mask bits -- and writes them once, so the kernel is
// bound by HBM for many rows and by one round of loads for one.  Vectors start
// at the 16-byte boundary at or before the row (the row's first and last
// vector go token by token); a row whose logits, history and output do not
// share such a boundary goes token by token throughout.
#include "common.cuh"

namespace nova {
namespace logits {

constexpr int THREADS = 256;
constexpr int VEC = 8;                  // tokens per thread
constexpr int CHUNK = THREADS * VEC;    // tokens per CTA, and per bias list

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

// Biases of a CTA's tokens up to this many go from lane to lane: each lane holds
// one, and a warp takes those of its own tokens.  More go through shared memory.
constexpr int FEW_BIASES = 64;

template <typename T>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(const Params p) {
    __shared__ __align__(16) float bias_s[CHUNK];
    const int row = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 31;
    const T* src = reinterpret_cast<const T*>(p.logits) + row * p.lstride;
    T* dst = reinterpret_cast<T*>(p.out) + row * p.ostride;
    const int16_t* hist = p.history ? p.history + row * p.hstride : nullptr;
    // Tokens before the row that its first vector would cover, and whether every pointer agrees on it.
    const int lead = int(hist ? reinterpret_cast<uintptr_t>(hist) / 2 % VEC : reinterpret_cast<uintptr_t>(src) / sizeof(T) % VEC);
    const bool vec = (reinterpret_cast<uintptr_t>(src) - lead * sizeof(T)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(dst) - lead * sizeof(T)) % 16 == 0;
    const int base = chunk * CHUNK - lead;                     // first token of this CTA
    if (base >= p.vocab) return;
    const int t0 = base + int(threadIdx.x) * VEC;
    const bool whole = vec && t0 >= 0 && t0 + VEC <= p.vocab;
    pdl_wait();

    // loads that nothing waits for, all in flight
    Vec<T> x;
    Vec<int16_t> h;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        x.v[i] = from_float<T>(0.f);
        h.v[i] = 0;
    }
    if (whole) {
        const uint4* s = reinterpret_cast<const uint4*>(src + t0);
#pragma unroll
        for (int i = 0; i < int(sizeof(x) / 16); ++i) reinterpret_cast<uint4*>(&x)[i] = s[i];
        if (hist) *reinterpret_cast<uint4*>(&h) = *reinterpret_cast<const uint4*>(hist + t0);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (t0 + i >= 0 && t0 + i < p.vocab) {
                x.v[i] = src[t0 + i];
                if (hist) h.v[i] = hist[t0 + i];
            }
    }
    int e0 = 0, e1 = 0;       // biases of this CTA's tokens: they lie in its list and, with a lead, in the one before
    if (p.bias_off) {
        const int* off = p.bias_off + int64_t(row) * p.chunks;
        e0 = off[min(max(chunk - (lead > 0), 0), p.chunks)];
        e1 = off[min(chunk + 1, p.chunks)];
    }
    const int which = !p.allowed ? -1 : p.allowed_row ? p.allowed_row[row] : row;
    const float rep = p.repetition ? p.repetition[row] : 1.f;
    const float inv = div_rn(1.f, rep);   // v * inv is within 2^-23 of v / rep, and no element waits for a division
    const float freq = p.frequency ? p.frequency[row] : 0.f;
    const float pres = p.presence ? p.presence[row] : 0.f;
    // 8 mask bits of this thread's tokens (all set: no mask)
    uint32_t keep = 0xFFu;
    if (which >= p.n_masks) {
        keep = 0u;
    } else if (which >= 0) {
        const uint32_t* m = p.allowed + which * p.mask_stride;
        const int f = max(t0, 0), words = (p.vocab + 31) / 32, w = f >> 5;
        const uint32_t lo = w < words ? m[w] : 0u;
        const uint32_t hi = (f & 31) > 32 - VEC && w + 1 < words ? m[w + 1] : 0u;
        keep = __funnelshift_r(lo, hi, f & 31) << (f - t0);
    }
    float b[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) b[i] = 0.f;
    const int count = e1 - e0;                                 // the same in the whole CTA
    if (count > 0 && count <= FEW_BIASES) {
        for (int e = e0; e < e1; e += 32) {
            const bool have = e + lane < e1;
            const int token = have ? p.bias_token[e + lane] : -1;
            const float value = have ? p.bias_value[e + lane] : 0.f;
            const int first = t0 - lane * VEC;                 // this warp's first token
            unsigned mine = __ballot_sync(0xffffffffu, have && token >= first && token < first + 32 * VEC);
            for (; mine; mine &= mine - 1) {
                const int l = __ffs(mine) - 1, k = __shfl_sync(0xffffffffu, token, l) - t0;
                const float v = __shfl_sync(0xffffffffu, value, l);
#pragma unroll
                for (int i = 0; i < VEC; ++i) b[i] = k == i ? v : b[i];
            }
        }
    } else if (count > 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) bias_s[i * THREADS + threadIdx.x] = 0.f;
        __syncthreads();
        for (int e = e0 + threadIdx.x; e < e1; e += THREADS) {
            const int at = p.bias_token[e] - base;
            if (at >= 0 && at < CHUNK) bias_s[at] = p.bias_value[e];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) b[i] = bias_s[int(threadIdx.x) * VEC + i];
    }
    Vec<T> y;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float v = to_float<T>(x.v[i]);
        const int hi = h.v[i], times = hi & 0x7FFF;
        v *= hi == 0 ? 1.f : v > 0.f ? inv : rep;
        // times as a float: in the mantissa of 2^23, which is subtracted (a conversion runs at a quarter of the rate)
        v -= times ? fmaf(freq, __int_as_float(0x4B000000 | times) - 8388608.f, pres) : 0.f;
        v += b[i];
        y.v[i] = from_float<T>((keep >> i) & 1u ? v : -INFINITY);
    }
    if (whole) {
        uint4* d = reinterpret_cast<uint4*>(dst + t0);
#pragma unroll
        for (int i = 0; i < int(sizeof(y) / 16); ++i) d[i] = reinterpret_cast<const uint4*>(&y)[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (t0 + i >= 0 && t0 + i < p.vocab) dst[t0 + i] = y.v[i];
    }
}

// A count or a prompt bit lives in half of a 32-bit word; both updates are
// whole-number atomics on that word, so their order does not matter.
__global__ void history_add_kernel(int16_t* history, int64_t stride, const int64_t* tokens, const int* off, int rows,
                                   int vocab, int prompt) {
    pdl_wait();
    const int row = blockIdx.y;
    const int64_t n = off ? off[row + 1] - off[row] : 1, first = off ? off[row] : row;
    for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x) {
        const int64_t t = tokens[first + i];
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
           static_cast<cudaStream_t>(stream), static_cast<int16_t*>(history), history_stride, tokens,
           static_cast<const int*>(off), int(rows), int(vocab), prompt);
    return check_launch("history add");
}
