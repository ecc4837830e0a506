// Attention over the 8-bit block-scaled cache for many query rows: prompts and long runs of tokens, on tcgen05.
//
// Same mathematics as the kernel for few rows: codes are exact in fp16, K's page scale multiplies the scores, V's goes
// into the probabilities. A unit is 256 query rows (128 at D = 256; token-major, the query heads of one kv head inside)
// of one sequence and kv head, as two tiles of 128; keys come 128 at a time, as eight 16-token tiles of whatever pages
// are seen. Per tile of rows:
//
//   S[128 x 128] = Q Kc^T     operands in shared memory, accumulator in tensor memory
//   P = 2^(S f - m) vs'       four warps, a thread per row: no shuffles; P goes back to tensor memory, over S, as two fp16
//                             numbers (22 bits, as in the kernel for few rows)
//   O[128 x D]  += P Vc       two products: P from tensor memory, Vc from shared memory, channels as its leading dimension
//
// Work is split by warps: 0 .. 3 and 4 .. 7 softmax and epilogue of the two tiles, 8 .. 11 load codes and write them as
// fp16 into the swizzled tiles (once for both), one thread of warp 12 issues the products. At 256 rows a byte of codes is
// worth 512 flops, so the tensor pipe (2 * 6 * 128 * 128 * D flops a step) and the exponentials (2 * 128 * 128, 16 a
// cycle) bound it, not HBM; one tile's products run under the other's exponentials. Every wait is bounded: a CTA whose
// wait gave up counts itself, waits for its products and leaves.
//
// Measured: 8 x 1024 query tokens behind 8192, 32/8 heads, no window: 1.65 ms, 624 TFLOP/s of the formula's 4 D flops a
// pair (e4m3 646), 0.37 and 0.38 of a large library product's rate, which the second product's half again is not counted
// in; head_dim 64: 381, 256 with 16/4 heads: 456. 2 x 1024 behind 6144, window 4096: 268 to 277 us in different runs, where
// the second round of 256 units leaves 40 of 148 multiprocessors idle: the tensor pipe is busy 35 % of the time, the
// exponentials' unit 31 %, the issue slots 41 %, so what bounds it is a tile's own chain (products, softmax, products).
// Steps of the softmax: two passes with the maximum 312 us -> none, packed arithmetic 288 -> masks as values 278 -> two
// tiles under one load of the keys 268. Two threads per row (274 us) and two CTAs of one tile (278) were no faster: with
// several roles' code in turn the instruction cache counts (the fully unrolled form took 343). The second half of P: 274 us
// without it, 321 with it while the next 32 scores were fetched under the present ones (84 to 108 bytes of spills a thread,
// twice the code in the loop), 267 since scores are fetched when they are due; an exponent for the tail 269, V's reference
// per row 272.
#include "q8_common.cuh"

namespace kivi {
namespace {

constexpr int kRows = 128, kKeys = 128, kThreads = 416;
constexpr float kMasked = -3.0e38f;    // score of a masked key, before its factor: 2^(factor * this) is 0 for factors of 1e-30 and more
constexpr float kHeadroomLog = 6.0f;   // log2(kQ8Headroom)
constexpr int kAtom = 128 * 128;   // bytes of 128 rows of 64 fp16 values, 128-byte swizzled

__device__ unsigned int g_q8_prompt_failures, g_q8_prompt_rejected;

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
    for (int it = 0; it < (1 << 17); ++it)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 128-byte-swizzled operand tiles: 8-row groups 1024 bytes apart. `lead`: bytes between 64-element column groups, which
// the layout asks for where the rows are the contraction (V: keys down, channels across).
__device__ __forceinline__ uint64_t operand(uint32_t smem, uint32_t lead) {
    return (uint64_t)((smem & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 with fp32 accumulator (bit 4), fp16 operands; bit 16: B's contraction runs down its rows; N >> 3, M >> 4
__host__ __device__ constexpr uint32_t shape(int n, bool b_rows) {
    return (1u << 4) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t (&v)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
          "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(at) : "memory");
}
// Loads wait in the same statement: nothing that uses the registers can be moved between the two.
__device__ __forceinline__ void load16(uint32_t at, uint32_t (&r)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void load32(uint32_t at, uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at) : "memory");
}
// two fp32 values in one instruction
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// What fp16 leaves of two values: x - h.x, y - h.y (exact in fp32), packed.
__device__ __forceinline__ uint32_t rest2(float x, float y, uint32_t h) {
    const unsigned short minus = 0xBC00;
    float lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tfma.rn.f32.f16 %0, a, %5, %3;\n\tfma.rn.f32.f16 %1, b, %5, %4;\n\t}"
        : "=f"(lo), "=f"(hi) : "r"(h), "f"(x), "f"(y), "h"(minus));
    return pack_half2(lo, hi);
}
__device__ __forceinline__ void store_wait() { __syncwarp(); asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Byte address of the 16-byte chunk `j` (8 values) of row `row` in a swizzled tile.
__device__ __forceinline__ uint32_t chunk_at(int row, int j) {
    return (uint32_t)((j >> 3) * kAtom + row * 128 + (((j & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ bool odd_half(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }

// Tiles of 128 rows per unit and stages of K and V: what shared memory (227 KB) and tensor memory (512 columns) hold.
template <int D>
constexpr int tiles_of() { return D == 256 ? 1 : 2; }
template <int D>
constexpr int stages_of() { return D == 256 ? 1 : 2; }
template <int D>
constexpr int smem_bytes() { return (tiles_of<D>() + 2 * stages_of<D>()) * kRows * D * 2 + 1024; }

template <int D, int FMT>
__global__ void __launch_bounds__(kThreads, 1) q8_prompt_kernel(const Q8AttnParams p) {
    constexpr int CPR = D / 16;            // 16-byte chunks of a row of codes
    constexpr int TILE = kRows * D * 2;    // bytes of an fp16 operand tile
    constexpr int TILES = tiles_of<D>(), STAGES = stages_of<D>();
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full_k[2], full_v[2], free_k[2], free_v[2], s_ready[2], p_ready[2], pv_done[2], drained;
    __shared__ uint32_t tmem_slot;
    // Of the steps in flight, per 16-token tile: the factor of its scores, log2 of V's scale, the first key; per step: first
    // and last key, the largest log2 of V's scale.
    // Four of them: K of step i is written when the products with K of step i - 2 are done, while the softmax may
    // still be at step i - 2; it is not at step i - 4, whose probabilities those products' order has waited for.
    __shared__ float meta_f[4][8], meta_lv[4][8], step_lv[4];
    __shared__ int meta_key0[4][8], step_key0[4], step_key1[4];
    __shared__ int odd_v, odd_page;        // a tail row held an infinity or NaN in V; a page's scale is NaN
    __shared__ uint32_t tail_top[4];       // largest finite magnitude in the tail's V, per loading warp
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkv = p.cache.nkv, block = 1 << p.cache.log2b;
    // the last rows first: without a window they have the most keys
    const int at_block = blockIdx.x % p.row_blocks;
    const Unit u = make_unit(p, blockIdx.x - at_block + (p.row_blocks - 1 - at_block), TILES * kRows);
    const int row_base = u.rb * TILES * kRows;
    if (u.counted && u.h == 0 && u.rb == 0 && tid == 0) atomicAdd(&g_q8_prompt_rejected, 1u);
    if (row_base >= u.rows) return;
    const View& v = u.v;
    const int steps = (u.items + 7) >> 3;
    const int tiles = row_base + kRows < u.rows ? TILES : 1;       // tiles with rows in them
    const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u, k_tile = smem + TILES * TILE, v_tile = k_tile + STAGES * TILE;

    if (tid == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mbar_init(&full_k[k], 128); mbar_init(&full_v[k], 128); mbar_init(&p_ready[k], 128);
            mbar_init(&free_k[k], 1); mbar_init(&free_v[k], 1); mbar_init(&s_ready[k], 1); mbar_init(&pv_done[k], 1);
        }
        mbar_init(&drained, 1);
        fence_barrier_init();
        odd_v = odd_page = 0;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int e = tid; e < tiles * kRows * (D / 8); e += kThreads) {   // query rows
        const int row = e / (D / 8), j = e % (D / 8), r = row_base + row;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (r < u.rows)
            x = *reinterpret_cast<const uint4*>(p.q + (long long)(u.row0 + r / p.qpk) * p.q_stride + (size_t)(u.h * p.qpk + r % p.qpk) * D + 8 * j);
        sts128(smem + (row >> 7) * TILE + chunk_at(row & 127, j), x);
    }
    fence_proxy_async();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
    auto tmem_s = [&](int t) { return tmem + t * kKeys; };
    auto tmem_o = [&](int t) { return tmem + TILES * kKeys + t * D; };
    bool failed = false;

    // row of a softmax thread
    const int t_mine = warp >> 2 & 1, r = row_base + t_mine * kRows + (tid & 127);
    const int hi = r < u.rows ? u.len - u.n + r / p.qpk : -1;
    const int lo = p.window == 0x7fffffff ? 0 : hi - p.window + 1;
    auto sees = [&](int key) { return key <= hi && (key >= lo || key < p.sinks); };

    if (warp < 8) {
        if (t_mine < tiles) {
        const uint32_t mine = (uint32_t)((warp & 3) * 32) << 16;   // this warp's lanes of tensor memory
        const uint32_t s_at = tmem_s(t_mine) + mine, o_at = tmem_o(t_mine) + mine;
        // P = 2^(s f - m) is kept below 2^8 by raising m when a sum says that it may not be: no pass over S for its maximum.
        // In fp16 it carries V's scale relative to 2^vref, an exponent not below any scale's that the row has met, and 2^6.
        // kQ8Unset: the row has met no key yet.
        float m = hi < 0 ? 0.0f : kQ8Unset, l = 0.0f, vref = -1000.0f;
        auto rescale_o = [&](float a) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                load16(o_at + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
                store16(o_at + c, o);
            }
        };
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
            const int b = i & 3;
            if (!wait_bar(&s_ready[t_mine], i & 1)) { failed = true; break; }
            fence_after();
            const int key0 = step_key0[b], key1 = step_key1[b];
            const bool masked = __any_sync(0xffffffffu, key1 > hi || (key0 < lo && key1 >= p.sinks));
            float lv = step_lv[b];
            if (__builtin_expect(masked, 0)) {      // of the tiles that this row sees
                lv = -1000.0f;
#pragma unroll 1
                for (int z = 0; z < 8; ++z) {
                    const int k0 = meta_key0[b][z];
                    if (k0 <= hi && (k0 + 15 >= lo || k0 < p.sinks)) lv = fmaxf(lv, meta_lv[b][z]);
                }
            }
            if (__builtin_expect(__any_sync(0xffffffffu, lv > vref), 0)) {   // O of the step before is complete, as S of this one is there
                const float next = lv > vref ? floorf(lv) + 1.0f : vref;
                if (i > 0) rescale_o(fast_exp2(vref - next));
                vref = next;
            }
            // 32 keys: scores to probabilities. What is rare is kept out of the way: this code is run over and over beside
            // two other roles' and its length counted more than its instructions.
            auto hide = [&](uint32_t (&s)[32], int c) {
                if (__builtin_expect(masked, 0)) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) if (!sees(meta_key0[b][2 * c + (e >> 4)] + (e & 15))) s[e] = __float_as_uint(kMasked);
                }
            };
            auto chunk = [&](uint32_t (&s)[32], int c) {
                hide(s, c);
                uint32_t out[16], rest[16];
                float sum;
                while (true) {
                    sum = 0.0f;
                    const float base = vref - kHeadroomLog + (m == kQ8Unset ? 0.0f : m);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float lw = meta_lv[b][2 * c + half], add = lw - base, f = meta_f[b][2 * c + half];
                        const uint64_t ff = pack2(f, f), aa = pack2(add, add);
                        uint64_t acc = pack2(0.0f, 0.0f);
#pragma unroll
                        for (int e = 16 * half; e < 16 * half + 16; e += 2) {
                            float x, y;
                            unpack2(fma2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), ff, aa), x, y);
                            x = fast_exp2(x);
                            y = fast_exp2(y);
                            acc = add2(acc, pack2(x, y));
                            out[e / 2] = pack_half2(x, y);
                            rest[e / 2] = rest2(x, y, out[e / 2]);   // takes the place of the scores, which are in tensor memory still
                        }
                        float x, y;
                        unpack2(acc, x, y);
                        sum = fmaf(x + y, fast_exp2(vref - kHeadroomLog - lw), sum);
                    }
                    if (__builtin_expect(!__any_sync(0xffffffffu, !(sum <= 256.0f) || m == kQ8Unset), 1)) break;
                    // the first keys of a row, or scores far above all before them
                    load32(s_at + 32 * c, s);
                    hide(s, c);
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (__uint_as_float(s[e]) != kMasked) top = fmaxf(top, __uint_as_float(s[e]) * meta_f[b][2 * c + (e >> 4)]);
                    // whole numbers: the factor is a power of two, and what is there already is not rounded again
                    const bool none = !__any_sync(0xffffffffu, top > m);
                    const float mn = fmaxf(m, ceilf(top)), a = fast_exp2(m - mn);
                    if (none) break;                    // nothing new to go by: NaN, or keys that nobody sees
                    // P of this step's earlier chunks, and O if it was rescaled in this step, are on their way to tensor
                    // memory: a load does not wait for an earlier store of the same columns by itself
                    store_wait();
                    m = mn;
                    l *= a;
                    if (i > 0) rescale_o(a);
#pragma unroll 1
                    for (int k = 0; k < c; ++k) {       // the chunks of P that are there already
                        uint32_t w[16], z[16];
                        load16(s_at + 32 * k, w);
                        load16(s_at + 32 * k + 16, z);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {   // in fp32: the factor alone may lie below fp16's range
                            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&z[e]));
                            const float x = (h.x + g.x) * a, y = (h.y + g.y) * a;
                            w[e] = pack_half2(x, y);
                            z[e] = rest2(x, y, w[e]);
                        }
                        store16(s_at + 32 * k, w);
                        store16(s_at + 32 * k + 16, z);
                    }
                }
                l += sum;
                store16(s_at + 32 * c, out);            // P in the place of the scores it came from
                store16(s_at + 32 * c + 16, rest);
            };
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t x[32];
                load32(s_at + 32 * c, x);
                chunk(x, c);
            }
            store_wait();
            fence_before();
            arrive(&p_ready[t_mine]);
        }
        if (!failed && steps > 0 && !wait_bar(&pv_done[t_mine], (steps - 1) & 1)) failed = true;
        fence_after();
        const float scale = l != 0.0f ? fast_exp2(vref - kHeadroomLog) / l : 0.0f;
        const size_t at = r < u.rows ? out_at(p, u, r, D) : 0;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t w[16];
            float o[16];
            if (steps > 0) load16(o_at + c, w);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = steps > 0 && l != 0.0f ? __uint_as_float(w[e]) * scale : 0.0f;
            if (r >= u.rows) {
                // a row behind the last: nothing to store
            } else if (p.out_h) {
#pragma unroll
                for (int e = 0; e < 16; e += 8)
                    *reinterpret_cast<uint4*>(p.out_h + at + c + e) = make_uint4(
                        pack_half2(o[e], o[e + 1]), pack_half2(o[e + 2], o[e + 3]), pack_half2(o[e + 4], o[e + 5]), pack_half2(o[e + 6], o[e + 7]));
            } else {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(p.out + at + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
        }
        }
    } else if (warp < 12) {
        const int c = tid - 256;
        const int sub_mask = (block >> 4) - 1, sub_log = p.cache.log2b - 4;
        const int* table = p.seq.tables + (size_t)u.seq * p.seq.width;
        int slot = q8_slot(p.seq, u.seq);
        if (!index_in_pool(slot, p.cache.num_slots)) {
            if (c == 0 && v.tail_tiles) atomicAdd(&g_q8_prompt_rejected, 1u);
            slot = 0;
        }
        auto tile_of = [&](int item) { return item < v.ns ? item : item - v.ns + v.w0; };
        auto unseen = [&](int key) { return key >= v.end || (key < v.low0 && key >= p.sinks); };
        // This thread's chunks: row16 and chunk of tile sub_of(k), k = 0 .. CPR - 1. Page codes are finite, so masked tokens'
        // rows may stay what they are; tail rows, which may hold anything, are fetched as zeros where nobody sees them.
        const int chunk = c % CPR;
        auto sub_of = [&](int k) { return D == 64 ? 2 * k + (c >> 6) : D == 128 ? k : k >> 1; };
        auto row_of = [&](int k) { return D == 64 ? (c >> 2) & 15 : D == 128 ? c >> 3 : (k & 1) * 8 + (c >> 4); };
        // lanes 0 .. 7 hold where the step's eight tiles start
        auto load_id = [&](int i) {
            const int item = 8 * i + (lane & 7);
            if (item >= v.tiles) return 0;
            const int page = tile_of(item) >> sub_log;
            return page < p.seq.width ? table[page] : -1;
        };
        // Codes travel ahead: a thread asks for its chunks of step i + 1 as soon as those of step i are stored (at D = 256,
        // where K's and V's together would not fit its registers, just before it waits for room in the tile).
        constexpr bool AHEAD = D < 256;
        uint4 x[2][CPR];
        auto fetch = [&](int which, int step, uint32_t start) {
            const uint8_t* codes = (which ? p.cache.v : p.cache.k) + chunk * 16;
            const int paged = v.tiles - 8 * step;
#pragma unroll
            for (int k = 0; k < CPR; ++k) {
                const uint32_t at = __shfl_sync(0xffffffffu, start, sub_of(k));
                x[which][k] = make_uint4(0u, 0u, 0u, 0u);
                if (sub_of(k) < paged) x[which][k] = __ldg(reinterpret_cast<const uint4*>(codes + (size_t)at * (16 * D) + row_of(k) * D));
            }
        };
        // id: of the step to come; where its tiles start, counted in tiles
        auto start_of = [&](int& id, int step) {
            if (!index_in_pool(id, p.cache.num_blocks)) {
                if (c < 8) atomicAdd(&g_q8_prompt_rejected, 1u);
                id = 0;
            }
            return ((uint32_t)id * nkv + u.h) * (uint32_t)(block >> 4) + (uint32_t)(tile_of(8 * step + (lane & 7)) & sub_mask);
        };
        int id = load_id(0), id_next = load_id(1);
        uint32_t start = start_of(id, 0);
        if (AHEAD) { fetch(0, 0, start); fetch(1, 0, start); }
        // The tail's V enters as a page's does: times a power of two that brings its largest value to 2^7 .. 2^8, whose log2
        // takes the place of the scale's. As it is, with scale 1, it would push the probabilities of pages of small values
        // in the same step below fp16's range.
        float tail_lv = -1000.0f, tail_mul = 1.0f;
        if (v.tail_tiles) {
            const __half* tail = p.cache.v_tail + ((size_t)slot * nkv + u.h) * block * D;
            uint32_t top = 0;
            for (int e = c; e < (v.end - v.paged) * (D / 8); e += 128) {
                if (unseen(v.paged + e / (D / 8))) continue;
                const uint4 y = *reinterpret_cast<const uint4*>(tail + (size_t)e * 8);
                const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t lo = w[k] & 0x7fffu, hi = w[k] >> 16 & 0x7fffu;
                    if (lo < 0x7c00u) top = max(top, lo);
                    if (hi < 0x7c00u) top = max(top, hi);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) tail_top[warp - 8] = top;
            asm volatile("bar.sync 1, 128;" ::: "memory");   // the loading warps
            top = max(max(tail_top[0], tail_top[1]), max(tail_top[2], tail_top[3]));
            if (top) {
                tail_lv = (float)(ilogbf(__half2float(__ushort_as_half((unsigned short)top))) - 7);
                tail_mul = exp2f(-tail_lv);
            }
        }
#pragma unroll 1
        for (int i = 0; i < steps && !failed; ++i) {
            const int first = 8 * i, b = i & 3, stage = i % STAGES;
            const int paged = min(8, max(0, v.tiles - first)), there = min(8, u.items - first);   // tiles of pages; of any kind
            float f = 1.0f, lv = -1000.0f;
            int key0 = 0x3fffffff;                       // a tile that is not there: no row sees that far
            if (c < paged) {
                float2 sc = p.cache.scales[(size_t)id * nkv + u.h];
                if (!(sc.x + sc.y == sc.x + sc.y)) { odd_page = 1; sc = make_float2(1.0f, 0.0f); }   // seen to at the end
                // a sum of products is below 2^33: times a factor as small as this it is 0, and kMasked times it still masks
                f = fmaxf(sc.x * p.scale_log2, 1e-30f);
                lv = sc.y == 0.0f ? -1000.0f : log2f(sc.y);
                key0 = tile_of(first + lane) * 16;
            } else if (c < there) {
                f = fmaxf(p.scale_log2, 1e-30f); lv = tail_lv;
                key0 = v.paged + (first + c - v.tiles) * 16;
            }
            const uint32_t start_now = start;
            id = id_next;
            id_next = load_id(i + 2);
            start = start_of(id, i + 1);
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                const uint32_t dst = (which ? v_tile : k_tile) + stage * TILE;
                if (!AHEAD) fetch(which, i, start_now);
                if (i >= STAGES && !wait_bar(which ? &free_v[stage] : &free_k[stage], (i / STAGES - 1) & 1)) { failed = true; break; }
                if (which == 0 && c < 32) {              // one warp: what the softmax has to know of the step
                    float lv_top = lv;
                    int k0 = key0, k1 = key0 + 15;
#pragma unroll
                    for (int z = 4; z > 0; z /= 2) {
                        lv_top = fmaxf(lv_top, __shfl_xor_sync(0xffffffffu, lv_top, z));
                        k0 = min(k0, __shfl_xor_sync(0xffffffffu, k0, z));
                        k1 = max(k1, __shfl_xor_sync(0xffffffffu, k1, z));
                    }
                    if (c < 8) {
                        meta_f[b][c] = f; meta_key0[b][c] = key0;
                        meta_lv[b][c] = lv == -1000.0f ? fmaxf(lv_top, -100.0f) : lv;
                    }
                    if (c == 0) { step_lv[b] = fmaxf(lv_top, -100.0f); step_key0[b] = k0; step_key1[b] = k1; }
                }
                // the two halves of a row's threads store in opposite order, so that eight threads meet eight bank groups
                const bool flip = chunk & 4;
#pragma unroll
                for (int k = 0; k < CPR; ++k) {
                    const int row = sub_of(k) * 16 + row_of(k);
                    const uint4 y = x[which][k];
                    const uint32_t w[4] = {flip ? y.z : y.x, flip ? y.w : y.y, flip ? y.x : y.z, flip ? y.y : y.w};
                    uint4 a, z;
                    q8_unpack<FMT>(w[0], a.x, a.y); q8_unpack<FMT>(w[1], a.z, a.w);
                    q8_unpack<FMT>(w[2], z.x, z.y); q8_unpack<FMT>(w[3], z.z, z.w);
                    sts128(dst + chunk_at(row, 2 * chunk + (flip ? 1 : 0)), a);
                    sts128(dst + chunk_at(row, 2 * chunk + (flip ? 0 : 1)), z);
                }
                if (there > paged) {                     // the step's tail tiles, over what was just written there
                    const __half* tail = (which ? p.cache.v_tail : p.cache.k_tail) + ((size_t)slot * nkv + u.h) * block * D;
#pragma unroll 1
                    for (int k = 0; k < CPR; ++k) {
                        if (sub_of(k) < paged || sub_of(k) >= there) continue;
                        const int row = sub_of(k) * 16 + row_of(k), at = (first + sub_of(k) - v.tiles) * 16 + row_of(k);
                        uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
                        if (!unseen(v.paged + at)) {
                            const uint4* src = reinterpret_cast<const uint4*>(tail + (size_t)at * D + chunk * 16);
                            const uint4 y = src[0], z = src[1];
                            w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w; w[4] = z.x; w[5] = z.y; w[6] = z.z; w[7] = z.w;
                        }
                        if (which) {   // 0 * infinity would reach rows that do not see the token: out, and seen to at the end
#pragma unroll
                            for (int z = 0; z < 8; ++z) {
                                if (odd_half(w[z])) odd_v = 1;
                                if ((w[z] & 0x7c00u) == 0x7c00u) w[z] &= 0xffff0000u;
                                if ((w[z] & 0x7c000000u) == 0x7c000000u) w[z] &= 0x0000ffffu;
                                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[z]));
                                w[z] = pack_half2(x.x * tail_mul, x.y * tail_mul);
                            }
                        }
                        sts128(dst + chunk_at(row, 2 * chunk), make_uint4(w[0], w[1], w[2], w[3]));
                        sts128(dst + chunk_at(row, 2 * chunk + 1), make_uint4(w[4], w[5], w[6], w[7]));
                    }
                }
                fence_proxy_async();
                arrive(which ? &full_v[stage] : &full_k[stage]);
                if (AHEAD) fetch(which, i + 1, start);
            }
        }
    } else if (lane == 0) {
        constexpr uint32_t qk = shape(kKeys, false), pv = shape(D, true);
        auto scores = [&](int t, int i) {
            const uint32_t q_at = smem + t * TILE, k_at = k_tile + (i % STAGES) * TILE;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {   // 16 channels: 32 bytes on in the swizzled row, the next 64 in the next atom
                const uint32_t at = (k >> 2) * kAtom + (k & 3) * 32;
                product_ss(tmem_s(t), operand(q_at + at, 16), operand(k_at + at, 16), qk, k > 0);
            }
            commit(&s_ready[t]);
            if (t == tiles - 1) commit(&free_k[i % STAGES]);
        };
        auto keys_there = [&](int i) {
            const bool ok = wait_bar(&full_k[i % STAGES], (i / STAGES) & 1);
            __threadfence_block();   // what the loading warps left beside the tile goes on to those that wait for s_ready
            fence_after();
            return ok;
        };
        failed = steps > 0 && !keys_there(0);
        for (int t = 0; t < tiles && steps > 0 && !failed; ++t) scores(t, 0);
        for (int i = 0; i < steps && !failed; ++i) {
            if (!wait_bar(&full_v[i % STAGES], (i / STAGES) & 1)) { failed = true; break; }
            for (int t = 0; t < tiles; ++t) {
                if (!wait_bar(&p_ready[t], i & 1)) { failed = true; break; }
                fence_after();
                const uint32_t v_at = v_tile + (i % STAGES) * TILE;
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k) {   // 16 keys: 8 columns of P, 8 of what fp16 left of it, 16 rows of V
                    const uint32_t p_at = tmem_s(t) + 32 * (k >> 1) + 8 * (k & 1);
                    product_ts(tmem_o(t), p_at, operand(v_at + 2048 * k, kAtom), pv, i > 0 || k > 0);
                    product_ts(tmem_o(t), p_at + 16, operand(v_at + 2048 * k, kAtom), pv, 1);
                }
                commit(&pv_done[t]);
                if (t == tiles - 1) commit(&free_v[i % STAGES]);
                if (i + 1 == steps) continue;
                // P gives way to the next S: the products that read it are done first
                if ((t == 0 && !keys_there(i + 1)) || !wait_bar(&pv_done[t], i & 1)) { failed = true; break; }
                fence_after();
                scores(t, i + 1);
            }
        }
        commit(&drained);
        if (!wait_bar(&drained, 0)) failed = true;
    }
    __syncwarp();
    fence_before();
    const bool cta_failed = __syncthreads_or(failed);
    if (warp == 12)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    if (cta_failed && tid == 0) atomicAdd(&g_q8_prompt_failures, 1u);
    if (odd_page && warp < 8 && t_mine < tiles && r < u.rows) {
        // rare: a row that sees a token of a page with a NaN scale yields NaN throughout
        const int* table = p.seq.tables + (size_t)u.seq * p.seq.width;
        const size_t at = out_at(p, u, r, D);
        for (int item = 0; item < v.tiles; ++item) {
            const int tile = item < v.ns ? item : item - v.ns + v.w0, page = tile >> (p.cache.log2b - 4);
            const int id = page < p.seq.width ? table[page] : 0;
            const float2 sc = p.cache.scales[(size_t)(index_in_pool(id, p.cache.num_blocks) ? id : 0) * nkv + u.h];
            if (sc.x + sc.y == sc.x + sc.y) continue;
            bool seen = false;
            for (int e = 0; e < 16; ++e) seen |= sees(tile * 16 + e);
            for (int ch = 0; seen && ch < D; ++ch) {
                if (p.out_h) p.out_h[at + ch] = __ushort_as_half((unsigned short)0x7fff);
                else p.out[at + ch] = __int_as_float(0x7fc00000);
            }
        }
    }
    if (odd_v && warp < 8 && t_mine < tiles && r < u.rows) {   // (one of a row's two threads)
        // rare: rows that see a tail token whose V holds an infinity or NaN yield NaN in that channel
        int slot = q8_slot(p.seq, u.seq);
        if (!index_in_pool(slot, p.cache.num_slots)) slot = 0;
        const __half* tail = p.cache.v_tail + ((size_t)slot * nkv + u.h) * block * D;
        const size_t at = out_at(p, u, r, D);
        for (int j = 0; v.paged + j < v.end; ++j) {
            if (!sees(v.paged + j)) continue;
            for (int ch = 0; ch < D; ++ch) {
                if ((__half_as_ushort(tail[(size_t)j * D + ch]) & 0x7c00u) != 0x7c00u) continue;
                if (p.out_h) p.out_h[at + ch] = __ushort_as_half((unsigned short)0x7fff);
                else p.out[at + ch] = __int_as_float(0x7fc00000);
            }
        }
    }
}

template <int D, int FMT>
cudaError_t launch(const Q8AttnParams& p, cudaStream_t stream) {
    auto kernel = q8_prompt_kernel<D, FMT>;
    static Q8SmemLimit limit;
    const cudaError_t e = limit.raise(kernel, smem_bytes<D>());
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)((size_t)p.seq.batch * p.cache.nkv * p.row_blocks), kThreads, smem_bytes<D>(), stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_q8_prompt(const Q8AttnParams& args, int d, int fmt, cudaStream_t stream) {
    Q8AttnParams p = args;
    const int rows = kRows * (d == 256 ? 1 : 2);
    p.row_blocks = (p.max_q * p.qpk + rows - 1) / rows;
    p.row_block0 = 0;
    const bool i8 = fmt == KIVI_Q8_INT8;
    switch (d) {
        case 64: return i8 ? launch<64, KIVI_Q8_INT8>(p, stream) : launch<64, KIVI_Q8_E4M3>(p, stream);
        case 128: return i8 ? launch<128, KIVI_Q8_INT8>(p, stream) : launch<128, KIVI_Q8_E4M3>(p, stream);
        default: return i8 ? launch<256, KIVI_Q8_INT8>(p, stream) : launch<256, KIVI_Q8_E4M3>(p, stream);
    }
}

cudaError_t q8_prompt_rejected(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_q8_prompt_rejected, sizeof(*count)); }
cudaError_t q8_prompt_failures(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_q8_prompt_failures, sizeof(*count)); }

}  // namespace kivi
