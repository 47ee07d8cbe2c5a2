// Attention of many query rows (prompt chunks) over the paged int8 cache on the
// 5th-generation tensor cores.
//
// 4 * 128 flops per (query row, key) and, at 100 rows or more, far fewer bytes:
// the tensor cores and the exponentials bound it (a 128 x 128 tile of scores is
// 1024 cycles of MMA and 1024 cycles of the 16 exponentials a cycle that an SM
// computes).  Measured: 2048 tokens x 32 heads over 30011 cached ones 975 us,
// 1.07 PFLOP/s; 509 over 8192 90 us and 7 for the join.  What bounds it is the
// chain within a 128-key step, about 4100 cycles with two halves in flight: 1480
// until the products are there, 590 to load the scores, 460 for their maximum,
// 2070 for the exponentials (the halves share 16 a cycle), 210 to store the
// weights.  Pairs of SMs sharing K and V lengthened it (1207 us), 64-key steps
// with two score buffers too (1285).
//
// One persistent CTA per SM walks segments of its own list: 256 query rows
// (token, query head of one KV head) of a request x a range of 64-token blocks,
// equal shares of the whole step's work for every CTA.  A step is 128 keys:
//   * warps 8-11 turn K and V codes into fp16(code * step + min) on their way
//     from global memory (the next step's codes and scales already in
//     registers) into two-stage 128-byte-swizzled shared-memory tiles -- the
//     same layout for both, read K-major as B of Q K^T and MN-major as B of P V;
//   * one thread issues tcgen05.mma: S_i = Q_i K^T and O_i += P_i V for the two
//     128-row halves i, so that one half's products run during the other
//     half's softmax; P_i comes from tensor memory, where it replaces S_i;
//   * warps 0-3 and 4-7 own one half each, a thread per row: running maximum and
//     sum in fp32, weights in fp16 (2^-11 of each, as the output's rounding).
//     The accumulator is rescaled only when a row's maximum has grown by more
//     than 2^8 since the last time: weights stay below 2^8, far from fp16's
//     range, and the factor cancels in O / l.
// A tile that was cut between CTAs leaves fp32 partials, joined in order by a
// second small kernel.  Every wait is bounded; after one that gave up the CTA
// stops, drains its MMAs and frees its tensor memory.
#include "paged.cuh"

namespace nova {
namespace paged {
namespace tc {

constexpr int THREADS = 512;           // 8 softmax warps, 4 loading warps, 1 MMA warp (and 3 idle ones: whole warpgroups)
// Registers per thread after the split: 256 x 160 + 128 x 144 + 128 x 48 = 65536, the 512 x 128 of the launch.
constexpr int REG_SOFTMAX = 160, REG_LOAD = 144, REG_MMA = 48;
static_assert(256 * REG_SOFTMAX + 128 * REG_LOAD + 128 * REG_MMA <= THREADS * 128, "register split");
constexpr int TILE = 32768;            // 128 rows x 128 channels fp16: two 64-channel halves of 16 KiB
constexpr int Q_OFF = 0, K_OFF = 2 * TILE, V_OFF = 4 * TILE;
constexpr int SMEM = 6 * TILE + 1024;
constexpr uint32_t S_COL = 0, O_COL = 256;   // tensor memory: S0 S1 O0 O1, 128 columns each

struct Params {
    const __half* q;
    int64_t q_t, q_h;
    const uint8_t* codes;
    const __half* scales;
    const __half* tails;
    __half* out;
    int64_t o_t, o_h;
    float* lse;
    const Seq* seqs;                   // the joining kernel's; segments carry what they need
    const int* pages;
    const TileSeg* segs;
    int* err;
    float* part;                       // [part][32][256][4]: four channels of all rows, then the next four
    float2* part_ml;
    int q_heads, kv_heads, gq, window;
    float scale_log2;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Two fp32 operations per instruction, and a three-way maximum: the softmax
// warps are bound by instruction issue as much as by the exponentials.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Low words of matrix descriptors in the 128-byte swizzle layout; the high word
// is the same for all: 8-row groups 1024 B apart (stride byte offset, [32,46)),
// version 1 [46,48), swizzle mode 2 = 128 B [61,64).  K-major: rows of 64 k.
// MN-major: rows of 64 MN elements, one row per k, the next 64 MN elements
// `mn_step` bytes on (leading byte offset, [16,30)).
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t kmajor(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t mnmajor(uint32_t saddr, uint32_t mn_step) {
    return ((saddr & 0x3FFFFu) >> 4) | ((mn_step >> 4) << 16);
}
// D[tmem] (+)= A B, A from shared memory / from tensor memory (fp16, kind::f16).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(DESC_HI)
        : "memory");
}

// Byte offset of 16-byte chunk c (0..15 along the channels) of row r in a tile.
__device__ __forceinline__ int tile_off(int r, int c) { return (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Codes and scales of one 64-token block that a loading thread holds: 8
// channels (chunk c = tid % 16) of rows tid / 16 + 8 i.
struct Raw {
    uint2 code[8];
    uint4 mn, st;
    int page;                          // -1: the open page, -2: nothing (zeros)
};

__device__ __forceinline__ uint4 dequant8(uint2 w, const uint4& st, const uint4& mn) {
    return make_uint4(hfma2(u8x2_lo_to_f16x2(w.x), st.x, mn.x), hfma2(u8x2_hi_to_f16x2(w.x), st.y, mn.y),
                      hfma2(u8x2_lo_to_f16x2(w.y), st.z, mn.z), hfma2(u8x2_hi_to_f16x2(w.y), st.w, mn.w));
}

__global__ void __launch_bounds__(THREADS, 1) paged_attn_tile_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], q_full[2], s_full[2], p_ready[2],
        o_full[2], drain;
    __shared__ uint32_t tmem_s;
    __shared__ int dead_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(smem);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&v_full[i], 4);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&q_full[i], 4);
        }
        mbar_init(&drain, 1);
        fence_mbar_init();
        dead_s = 0;
    }
    if (warp == 12) {
        tmem_alloc(&tmem_s, 512);
        tmem_relinquish();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    volatile int* dead = &dead_s;
    // A bounded wait; false once any wait of this CTA has given up.
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
        if (mbar_wait(bar, parity, p.err, 2)) return true;
        *dead = 1;
        return false;
    };
    pdl_wait();

    if (warp >= 8 && warp < 12) {
        // ------------------------------------------------ loading warps
        reg_inc<REG_LOAD>();
        const int tid = threadIdx.x - 256, c = tid & 15, r0 = tid >> 4;   // 8 channels, first row (of 8)
        uint32_t kc = 0;               // steps so far
        for (int sg = blockIdx.x; sg >= 0;) {
            const TileSeg it = p.segs[sg];
            sg = it.next;
            const int n_full = it.kv_len / PT;
            const int steps = (it.blk1 - it.blk0 + 1) >> 1;
            const int* pages = p.pages + it.page_off;
            const uint8_t* codes = p.codes + it.head * 2 * HALF_ROW + r0 * D + 8 * c;
            const __half* scales = p.scales + it.head * 4 * D + 8 * c;
            const int code_step = p.kv_heads * 2 * HALF_ROW, scale_step = p.kv_heads * 4 * D;   // per page
            // Page number of the segment's block b (-1: the open page, -2: past the end).  Lane b % 32 holds
            // those of 32 blocks, the next 32 already requested: nothing waits for a page number.
            auto lookup = [&](int b) { return it.blk0 + b < min(it.blk1, n_full) ? pages[it.blk0 + b] : -1; };
            int ids = lookup(lane), ids_next = lookup(32 + lane);
            auto page_of = [&](int b) {
                const int id = __shfl_sync(0xffffffffu, ids, b & 31);
                return it.blk0 + b < it.blk1 ? id : -2;
            };
            auto fetch = [&](Raw& raw, int page, int j) {
                raw.page = page;
                if (page >= 0) {
                    const uint8_t* src = codes + int64_t(page) * code_step + j * HALF_ROW;
                    const __half* sc = scales + int64_t(page) * scale_step + j * 2 * D;
#pragma unroll
                    for (int i = 0; i < 8; ++i) raw.code[i] = *reinterpret_cast<const uint2*>(src + 8 * i * D);
                    raw.mn = *reinterpret_cast<const uint4*>(sc);
                    raw.st = *reinterpret_cast<const uint4*>(sc + D);
                }
            };
            auto store = [&](const Raw& raw, uint32_t tile, int half, int j) {
                const uint32_t dst = tile + half * 8192 + tile_off(r0, c);   // 8 rows on: 1024 bytes, the same swizzle
                if (raw.page >= 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sts128(dst + i * 1024, dequant8(raw.code[i], raw.st, raw.mn));
                } else {               // the open page (slots that hold no token read as zero) or nothing
                    const __half* src = p.tails + half_off(it.tail, p.kv_heads, it.head, j) + 8 * c;
                    const int live = raw.page == -1 ? it.kv_len - n_full * PT : 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = r0 + 8 * i;
                        sts128(dst + i * 1024,
                               r < live ? *reinterpret_cast<const uint4*>(src + r * D) : make_uint4(0u, 0u, 0u, 0u));
                    }
                }
            };
            auto publish = [&](uint64_t* bar) {
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            Raw k0, k1, v0, v1;
            int pg0 = it.page[0], pg1 = it.blk0 + 1 < it.blk1 ? it.page[1] : -2;
            fetch(k0, pg0, 0);
            fetch(k1, pg1, 0);
            fetch(v0, pg0, 1);
            fetch(v1, pg1, 1);
            bool ok = true;
            for (int j = 0; j < steps; ++j, ++kc) {
                const uint32_t st = kc & 1u, ph = ((kc >> 1) & 1u) ^ 1u;
                if (kc >= 2 && !(ok = wait(&k_empty[st], ph))) break;
                store(k0, sbase + K_OFF + st * TILE, 0, 0);
                store(k1, sbase + K_OFF + st * TILE, 1, 0);
                publish(&k_full[st]);
                const int b = 2 * j + 2;
                if ((b & 31) == 0) {
                    ids = ids_next;
                    ids_next = lookup(b + 32 + lane);
                }
                pg0 = page_of(b);
                pg1 = page_of(b + 1);
                fetch(k0, pg0, 0);
                fetch(k1, pg1, 0);
                if (kc >= 2 && !(ok = wait(&v_empty[st], ph))) break;
                store(v0, sbase + V_OFF + st * TILE, 0, 1);
                store(v1, sbase + V_OFF + st * TILE, 1, 1);
                publish(&v_full[st]);
                fetch(v0, pg0, 1);
                fetch(v1, pg1, 1);
            }
            if (!ok) break;
        }
    } else if (warp >= 12) {
        // ------------------------------------------------ MMA issue
        reg_dec<REG_MMA>();
        if (warp == 12) {              // the whole warp walks along, so that addresses stay in uniform registers
            constexpr uint32_t idesc_qk = tc_idesc_f16(128, 128);
            constexpr uint32_t idesc_pv = tc_idesc_f16(128, 128) | (1u << 16);   // B MN-major
            uint32_t kc = 0, sc[2] = {0u, 0u}, pc[2] = {0u, 0u};   // steps; segments and steps of each half
            bool ok = true;
            auto qk = [&](int i, uint32_t st) {
                const uint32_t a = kmajor(sbase + Q_OFF + i * TILE), b = kmajor(sbase + K_OFF + st * TILE);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t step = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                        mma_ss(tmem + S_COL + i * 128, a + step, b + step, idesc_qk, k > 0);
                    }
                    tc_commit(&s_full[i]);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (elect_one()) tc_commit(bar);
                __syncwarp();
            };
            for (int sg = blockIdx.x; sg >= 0 && ok;) {
                const TileSeg it = p.segs[sg];
                sg = it.next;
                const int steps = (it.blk1 - it.blk0 + 1) >> 1, halves = it.nrows > 128 ? 2 : 1;
                if (!(ok = wait(&k_full[kc & 1u], (kc >> 1) & 1u))) break;
                for (int i = 0; i < halves; ++i) {
                    if (!(ok = wait(&q_full[i], sc[i]++ & 1u))) break;
                    qk(i, kc & 1u);
                }
                if (!ok) break;
                commit(&k_empty[kc & 1u]);
                for (int j = 0; j < steps && ok; ++j, ++kc) {
                    const uint32_t st = kc & 1u;
                    if (!(ok = wait(&v_full[st], (kc >> 1) & 1u))) break;
                    for (int i = 0; i < halves; ++i) {
                        if (!(ok = wait(&p_ready[i], pc[i] & 1u))) break;
                        ++pc[i];
                        tc_fence_after();
                        const uint32_t b = mnmajor(sbase + V_OFF + st * TILE, 16384);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                mma_ts(tmem + O_COL + i * 128, tmem + S_COL + i * 128 + 8 * k, b + (k * 2048 >> 4), idesc_pv,
                                       j > 0 || k > 0);
                            if (j + 1 == steps) tc_commit(&o_full[i]);
                        }
                        __syncwarp();
                        if (j + 1 < steps) {
                            const uint32_t n = kc + 1;
                            if (i == 0 && !(ok = wait(&k_full[n & 1u], (n >> 1) & 1u))) break;
                            qk(i, n & 1u);
                        }
                    }
                    if (!ok) break;
                    commit(&v_empty[st]);
                    if (j + 1 < steps) commit(&k_empty[(kc + 1) & 1u]);
                }
            }
            commit(&drain);            // every MMA of this CTA has completed before its tensor memory is freed
            mbar_wait(&drain, 0u, p.err, 3);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax warps
        reg_inc<REG_SOFTMAX>();
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;    // row of the half = tensor memory lane
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + S_COL + half * 128 + lanes, o_addr = tmem + O_COL + half * 128 + lanes;
        uint32_t sc = 0, oc = 0;       // steps and segments of this half so far
        bool ok = true;
        // The CTA's first segment from sg on that has rows in this half.
        auto next_seg = [&](int sg) {
            while (sg >= 0 && p.segs[sg].nrows <= half * 128) sg = p.segs[sg].next;
            return sg;
        };
        // This warp's 32 rows of a segment's Q into shared memory, two rows per load (a row per lane was 32 cache lines
        // a load: 5500 cycles until the tile was there, 2700 this way).  Rows past the segment's repeat its last one and
        // are not stored.  Called when every score of this half's last segment is complete, so its tile is free.
        auto load_q = [&](const TileSeg& it) {
            const int arow = it.row0 + min(half * 128 + row, it.nrows - 1), tok = arow / p.gq;
            const int64_t off = int64_t(it.q_start + tok) * p.q_t + int64_t(it.head * p.gq + arow - tok * p.gq) * p.q_h;
            const int c = lane & 15, r0 = lane >> 4;
            uint4 v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                v[i] = *reinterpret_cast<const uint4*>(p.q + __shfl_sync(0xffffffffu, off, 2 * i + r0) + 8 * c);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sts128(sbase + Q_OFF + half * TILE + tile_off((warp & 3) * 32 + 2 * i + r0, c), v[i]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[half]);
        };
        int sg = next_seg(blockIdx.x);
        if (sg >= 0) load_q(p.segs[sg]);
        while (sg >= 0 && ok) {
            const TileSeg it = p.segs[sg];
            const int start = it.start, steps = (it.blk1 - it.blk0 + 1) >> 1;
            const int r = half * 128 + row;                          // row of the segment
            const bool live = r < it.nrows;
            const int arow = it.row0 + (live ? r : it.nrows - 1), tok = arow / p.gq, pos = start + tok;
            const int head = it.head * p.gq + arow - tok * p.gq;
            const int first_pos = start + (it.row0 + half * 128) / p.gq;
            const int last_pos = start + (it.row0 + min(half * 128 + 127, it.nrows - 1)) / p.gq;
            float m = -INFINITY, l = 0.f;                            // m: the maximum that O and l are relative to (log2)
            for (int j = 0; j < steps; ++j, ++sc) {
                const int key0 = (it.blk0 + 2 * j) * PT;
                if (!(ok = wait(&s_full[half], sc & 1u))) break;
                tc_fence_after();
                float x[128];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld32(s_addr + 32 * k, x + 32 * k);
                tmem_wait_ld();
                if (key0 + 127 > first_pos || (p.window > 0 && key0 <= last_pos - p.window)) {
                    const int hi = pos - key0, lo = p.window > 0 ? hi - p.window : -1;   // keys lo < k <= hi
#pragma unroll
                    for (int k = 0; k < 128; ++k) x[k] = k <= hi && k > lo ? x[k] : -INFINITY;
                }
                float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int k = 4; k < 124; k += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[k + 2 * e], x[k + 2 * e + 1]);
                mx[0] = max3(mx[0], x[124], x[125]);
                mx[1] = max3(mx[1], x[126], x[127]);
                const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;
                const bool grow = top > m + 8.f;
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, grow)) {          // O of the previous steps is complete: s_full says so
                    const float m_new = grow ? top : m;
                    const float alpha = grow ? ex2(m - m_new) : 1.f;
                    m = m_new;
                    l *= alpha;
#pragma unroll
                    for (int k = 0; k < 128; k += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + k, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st16(o_addr + k, o);
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), base2 = make_float2(-base, -base);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 y = fma2(make_float2(x[32 * h + 2 * k], x[32 * h + 2 * k + 1]), scale2, base2);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        sum[k & 1] = add2(sum[k & 1], y);
                        w[k] = pack_f16x2(y.x, y.y);
                    }
                    tmem_st16(s_addr + 16 * h, w);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[half]);
            }
            if (!ok) break;
            // the next segment's Q: its first scores are computed while this one's result is stored
            sg = next_seg(it.next);
            if (sg >= 0) load_q(p.segs[sg]);
            if (!(ok = wait(&o_full[half], oc & 1u))) break;
            ++oc;
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            __half* dst = p.out + int64_t(it.q_start + tok) * p.o_t + int64_t(head) * p.o_h;
            float4* prow = reinterpret_cast<float4*>(p.part) + int64_t(it.part) * 32 * 256 + r;
#pragma unroll
            for (int k = 0; k < 128; k += 32) {
                float o[32];
                tmem_ld32(o_addr + k, o);
                tmem_wait_ld();
                if (!live) continue;
                if (it.part < 0) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(dst + k + e) =
                            make_uint4(pack_f16x2(o[e] * inv, o[e + 1] * inv), pack_f16x2(o[e + 2] * inv, o[e + 3] * inv),
                                       pack_f16x2(o[e + 4] * inv, o[e + 5] * inv), pack_f16x2(o[e + 6] * inv, o[e + 7] * inv));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        prow[(k + e) * 64] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live) {
                if (it.part >= 0)
                    p.part_ml[int64_t(it.part) * 256 + r] = make_float2(m, l);
                else if (p.lse)
                    p.lse[int64_t(it.q_start + tok) * p.q_heads + head] =
                        l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
            }
            tc_fence_before();         // the next segment's first product overwrites O after this half's next p_ready
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partials of tiles that were cut, in segment order.  A CTA takes 32
// rows, a lane one row and a warp 4 * C channels: partials are read as they were
// written, 512 consecutive bytes per warp and load, eight or more loads in flight.
// Few joins have many parts each and want all SMs at once (C = 1: 17 parts of 8
// tiles take 8.1 us, 12.5 with C = 4); many joins fill the SMs by themselves and
// want whole sectors written and few CTAs (C = 4: 64 tiles of 2 parts take 6.7 us,
// 11 with C = 1).
template <int C>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const Params p, const TileJoin* joins) {
    pdl_wait();
    const TileJoin it = joins[blockIdx.x];
    const int r = int(blockIdx.y) * 32 + int(threadIdx.x & 31), c = (int(blockIdx.z) * 8 + int(threadIdx.x >> 5)) * C;
    if (r >= it.nrows) return;
    const float2* ml = p.part_ml + int64_t(it.part0) * 256 + r;
    const float4* part = reinterpret_cast<const float4*>(p.part) + (int64_t(it.part0) * 32 + c) * 256 + r;
    float M = -INFINITY, L = 0.f;
#pragma unroll 8
    for (int k = 0; k < it.n_parts; ++k) M = fmaxf(M, ml[k * 256].x);
    float4 o[C] = {};
#pragma unroll C == 1 ? 8 : 2
    for (int k = 0; k < it.n_parts; ++k) {
        const float2 e = ml[k * 256];
        float4 a[C];
        for (int j = 0; j < C; ++j) a[j] = part[(int64_t(k) * 32 + j) * 256];
        const float wt = M == -INFINITY ? 0.f : exp2f(e.x - M);
        L += wt * e.y;
        for (int j = 0; j < C; ++j) {
            o[j].x += wt * a[j].x; o[j].y += wt * a[j].y; o[j].z += wt * a[j].z; o[j].w += wt * a[j].w;
        }
    }
    const Seq s = p.seqs[it.seq];
    const int row = it.row0 + r, tok = row / p.gq, head = it.head * p.gq + row - tok * p.gq;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    for (int j = 0; j < C; ++j)
        *reinterpret_cast<uint2*>(p.out + int64_t(s.q_start + tok) * p.o_t + int64_t(head) * p.o_h + 4 * (c + j)) =
            make_uint2(pack_f16x2(o[j].x * inv, o[j].y * inv), pack_f16x2(o[j].z * inv, o[j].w * inv));
    if (p.lse && c == 0)
        p.lse[int64_t(s.q_start + tok) * p.q_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace tc

int launch_tiles(const nova_paged_attn_args* a, const nova_paged_plan_info* info, const nova_paged_schedule& s,
                 cudaStream_t stream) {
    tc::Params p{};
    p.q = static_cast<const __half*>(a->q);
    p.q_t = a->q_t_stride;
    p.q_h = a->q_h_stride;
    p.codes = static_cast<const uint8_t*>(a->codes);
    p.scales = static_cast<const __half*>(a->scales);
    p.tails = static_cast<const __half*>(a->tails);
    p.out = static_cast<__half*>(a->out);
    p.o_t = a->o_t_stride;
    p.o_h = a->o_h_stride;
    p.lse = static_cast<float*>(a->lse);
    p.seqs = reinterpret_cast<const Seq*>(a->plan + info->seq_off);
    p.pages = a->plan + info->page_off;
    p.segs = reinterpret_cast<const TileSeg*>(a->plan + s.segs_off);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.err = reinterpret_cast<int*>(ws);
    p.part = reinterpret_cast<float*>(ws + s.tile_parts_off);
    p.part_ml = reinterpret_cast<float2*>(p.part + s.n_tile_parts * 256 * D);
    p.q_heads = int(info->q_heads);
    p.kv_heads = int(info->kv_heads);
    p.gq = p.q_heads / p.kv_heads;
    p.window = int(s.window);
    p.scale_log2 = float(a->scale * 1.4426950408889634);
    static bool ready[kMaxDevices];        // shared-memory limit raised on this device
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices || !ready[dev]) {
        if (cudaFuncSetAttribute(reinterpret_cast<const void*>(&tc::paged_attn_tile_kernel),
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, tc::SMEM) != cudaSuccess)
            return check_launch("paged attention");
        if (dev >= 0 && dev < kMaxDevices) ready[dev] = true;
    }
    launch(tc::paged_attn_tile_kernel, dim3(unsigned(s.n_ctas)), dim3(tc::THREADS), tc::SMEM, stream, p);
    if (int rc = check_launch("paged attention")) return rc;
    if (!s.n_joins) return NOVA_OK;
    const bool few = s.n_joins <= 16;  // fewer CTAs of 8 per join than SMs
    launch(few ? tc::paged_attn_join_kernel<1> : tc::paged_attn_join_kernel<4>, dim3(unsigned(s.n_joins), 8, few ? 4 : 1),
           dim3(256), 0, stream, p, reinterpret_cast<const TileJoin*>(a->plan + s.joins_off));
    return check_launch("paged attention");
}

}  // namespace paged
}  // namespace nova
