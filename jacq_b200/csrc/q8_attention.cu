// Attention over the 8-bit block-scaled cache: one query token per sequence (serving), short runs and prompts.
//
//   s_ij = scale * ks(page of j) * (q_i . kc_j),  out_i = sum_j p_ij vs(page of j) vc_j / sum_j p_ij,  p = 2^(s log2e - m)
//
// kc, vc are codes: both formats are exact in fp16, and a page has ONE scale, so neither K nor V is ever scaled element
// by element: K's scale multiplies the 16 x rows score tile, V's goes into the probabilities. The products run on
// mma.sync m16n8k16 with tokens (QK) and channels (PV) as the 16 side and the query rows as the 8 side. What bounds a
// single-token call is HBM: 2 D bytes per token and kv head against 4 D flops per query row.
//
// The order of the contraction index is free, and so is the order of the output channels, so lane (g, t) = (lane / 4,
// lane % 4) takes of a 16-token tile the bytes its fragments need in 16-byte pieces: K rows g and g + 8, channels
// 16 (t + 4 j) ..; V tokens 2t, 2t+1, 2t+8, 2t+9, channels (D / 8) g .. . The warp copies a tile as whole 128-byte lines
// into its own ring (copying the pieces straight to the lanes that use them, in half lines, capped the kernel at
// 5.0 TB/s however many warps there were), under a swizzle that frees the reads of bank conflicts; cp.async groups and
// __syncwarp are the only synchronisation.
//
// A sequence's context is cut into `parts`, one CTA each, chosen by the model at plan_parts. Few parts of few units form
// a thread-block cluster and join through distributed shared memory; others leave partials for a merge kernel that is
// launched early. With page masses every tile leaves its rows' sums and the maxima they refer to (8 bytes per row and 16
// tokens), and the join adds them to the masses once the final maximum and sum are known: no atomics, a fixed order.
//
// Measured (device time): 128 x 8192 tokens, 32/8 heads, int8: 349 us, 6.1 TB/s, 0.95 of the copy rate; back to back at
// the power limit 404 us, where the time follows the instructions. One context of 32768 tokens, 40/8 heads, with
// masses: 28 us (10 us of data: start, join and 2 us a launch are what remains). 4 x 512 tokens, 32/4 heads of 64: 6.8 us.
// Steps: pieces copied to the lanes that use them 528 us -> whole lines 363 -> two tiles at a time 350 -> whole
// contexts in two parts 347 -> second halves of the probabilities 354 -> in the same product 349.
#include <cooperative_groups.h>
#include <type_traits>

#include "q8_common.cuh"

namespace kivi {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxParts = 32;

__device__ unsigned int g_q8_attn_rejected;

// mma16816 without "volatile": the products may be moved among the unpacking
__device__ __forceinline__ void product(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D>
struct Tile {
    static constexpr int KC = D / 64;            // 16-byte pieces of a K row per lane
    static constexpr int MT = D / 16;            // channel tiles of the output
    static constexpr int VP = D == 256 ? 2 : 1;  // pieces of a V row per lane
    static constexpr int VB = D == 64 ? 8 : 16;  // bytes of a piece
    static constexpr int VW = VB / 4;            // words (4 channels) of a piece
    static constexpr int BYTES = 16 * D;         // K or V codes of a tile
    static constexpr int CPR = D / 16;           // 16-byte chunks of a row
    static constexpr int STAGE = 2 * BYTES + 16; // K, V, scales
    // A row's chunks are stored under an exclusive or with a function of the row, so that the reads below spread over
    // the banks: K reads touch rows g and chunks t + 4 j, V reads rows 2 t .. and chunks g.
    static __device__ __forceinline__ int k_swizzle(int row) { return D == 64 ? 0 : (row & 1) << 2; }
    static __device__ __forceinline__ int v_swizzle(int row) { return D == 64 ? (row >> 1) & 3 : ((row >> 1) & 3) << 1; }
};

// Channel of output tile mt, half hf (rows g / g + 8 of the fragment) on lanes of group g.
template <int D>
__device__ __forceinline__ int channel_of(int g, int mt, int hf) {
    if constexpr (D == 256) return (mt < 8 ? 0 : 128) + 16 * g + 2 * (mt & 7) + hf;
    else return (D / 8) * g + 2 * mt + hf;
}

// Where row r, channel ch (even) lies among the accumulators, [accumulator][lane].
template <int D>
__device__ __forceinline__ int accumulator_of(int r, int ch) {
    const int g = D == 256 ? (ch & 127) >> 4 : ch / (D / 8), in = D == 256 ? ch & 15 : ch % (D / 8);
    const int mt = (D == 256 ? (ch >> 7) * 8 : 0) + (in >> 1);
    return (((r >> 3) * (D / 16) + mt) * 4 + 2 * (in & 1) + (r & 1)) * 32 + g * 4 + ((r >> 1) & 3);
}

__device__ __forceinline__ void store8(const Q8AttnParams& p, size_t at, const float (&x)[8]) {
    if (p.out_h) {
        *reinterpret_cast<uint4*>(p.out_h + at) =
            make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
    } else {
        *reinterpret_cast<float4*>(p.out + at) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p.out + at + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// Adds to the masses of pages first, first + step, ...: page p's tiles, whichever part met them, relative to the unit's
// final maximum f_m and 1 / sum f_il of every row.
template <int R>
__device__ __forceinline__ void add_masses(const Q8AttnParams& p, const Unit& u, const float* f_m, const float* f_il, int first, int step) {
    const int sub_log = p.cache.log2b - 4, subs = 1 << sub_log;
    const int pages = (u.len + (1 << p.cache.log2b) - 1) >> p.cache.log2b;
    const float2* ws = p.page_ws + (size_t)(u.seq * p.cache.nkv + u.h) * p.ws_tiles * R;
    float* mass = p.mass + ((size_t)u.seq * p.cache.nkv + u.h) * p.mass_width;
    for (int page = first; page < pages; page += step) {
        float sum = 0.0f;
        const int t0 = page << sub_log;
        for (int k = 0; k < subs; ++k) {
            int item;
            if (t0 * 16 < u.v.paged) {
                const int tile = t0 + k;
                if (tile < u.v.ns) item = tile;
                else if (tile >= u.v.w0 && tile - u.v.w0 + u.v.ns < u.v.tiles) item = tile - u.v.w0 + u.v.ns;
                else continue;
            } else {
                if (k >= u.v.tail_tiles) break;
                item = u.v.tiles + k;
            }
            float2 x[R];
#pragma unroll
            for (int r = 0; r < R; ++r) x[r] = __ldcg(ws + (size_t)item * R + r);
#pragma unroll
            for (int r = 0; r < R; ++r) sum += x[r].x * fast_exp2(x[r].y - f_m[r]) * f_il[r];
        }
        if (sum != 0.0f) mass[page] += sum;
    }
}

// Two shapes of the kernel. Four warps and a shallow ring, several CTAs per multiprocessor, where there are units enough
// to fill it; eight warps and a deep ring, one CTA per multiprocessor, where there are few and each warp's own copies
// have to cover the latency.
constexpr int tiles_at_once(int d) { return d == 256 ? 1 : 2; }
template <int D, int kWarps>
constexpr int stages_of() { return kWarps == 4 ? (D == 64 ? 3 : D == 128 ? 2 : 3) : D == 64 ? 5 : 3; }
template <int D, int kWarps>
constexpr int ctas_of() { return kWarps == 8 ? 1 : D == 64 ? 4 : D == 128 ? 3 : 2; }

// Query rows of a unit: at most 4, at most 8, at most 16. Probabilities are kept to 22 bits as two fp16 numbers (the
// output's own rounding is then the only one of its size; one number alone gave 1.4 times the plain form's error). With
// at most 4 rows the second numbers are columns 4 .. 7 of the same product, whose queries repeat columns 0 .. 3; beyond
// that they take a second product. 128 x 8192 tokens, 4 rows, back to back at the power limit: 408 us with one number,
// 404 with both in one product, 419 with two products.
constexpr int kRows4 = 4, kRows8 = 8, kRows16 = 16;

template <int D, int FMT, int ROWS, bool MASS, int kWarps, int NT>   // NT: groups of 8 columns, ROWS / 8 or 1
__global__ void __launch_bounds__(kWarps * 32, ctas_of<D, kWarps>()) q8_attention_kernel(const Q8AttnParams p) {
    constexpr bool FOLD = ROWS == kRows4;
    using T = Tile<D>;
    constexpr int R = 8 * NT, S = stages_of<D, kWarps>(), TPI = tiles_at_once(D);
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    __shared__ float c_m[R], c_l[R];             // this CTA's merged state, read by its cluster
    __shared__ float f_m[R], f_il[R];            // the unit's final maximum and 1 / sum
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int nkv = p.cache.nkv, block = 1 << p.cache.log2b;
    const int part = blockIdx.x % p.parts, unit = blockIdx.x / p.parts;
    const Unit u = make_unit(p, unit, R);
    const int seq = u.seq, h = u.h, rb = u.rb, len = u.len, n = u.n, row0 = u.row0, rows = u.rows, items = u.items;
    const View& v = u.v;
    if (u.counted && h == 0 && rb == 0 && part == 0 && threadIdx.x == 0) atomicAdd(&g_q8_attn_rejected, 1u);
    if (rb * R >= rows) return;                  // uniform over the cluster
    const int i0 = min(part * p.chunk, items), i1 = min(i0 + p.chunk, items);
    if (p.cluster == 0 && i0 == i1 && part > 0) return;   // the merge knows how many parts have something

    // ---- query rows as B fragments, in the channel order of the K pieces
    uint32_t qf[NT][T::MT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = rb * R + 8 * nt + (FOLD ? g & 3 : g);
        const __half* row = p.q + (long long)(row0 + r / p.qpk) * p.q_stride + (size_t)(h * p.qpk + r % p.qpk) * D + 16 * t;
#pragma unroll
        for (int j = 0; j < T::KC; ++j) {
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            if (r < rows) {
                a = *reinterpret_cast<const uint4*>(row + 64 * j);
                b = *reinterpret_cast<const uint4*>(row + 64 * j + 8);
            }
            qf[nt][4 * j][0] = a.x; qf[nt][4 * j][1] = a.y; qf[nt][4 * j + 1][0] = a.z; qf[nt][4 * j + 1][1] = a.w;
            qf[nt][4 * j + 2][0] = b.x; qf[nt][4 * j + 2][1] = b.y; qf[nt][4 * j + 3][0] = b.z; qf[nt][4 * j + 3][1] = b.w;
        }
    }
    // keys that the lane's score columns (rows 2t, 2t + 1 of each 8) see
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = rb * R + 8 * nt + (FOLD ? 2 * (t & 1) : 2 * t) + c;
            hi[nt][c] = r < rows ? len - n + r / p.qpk : -1;
            lo[nt][c] = p.window == 0x7fffffff ? 0 : hi[nt][c] - p.window + 1;
        }

    float o[NT][T::MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < T::MT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
        m[nt][0] = m[nt][1] = kQ8Unset;
        l[nt][0] = l[nt][1] = 0.0f;
    }
    // V's scales enter the fp16 probabilities relative to vref, a power of two not below any met so far (0: none yet). One
    // for all columns: where rows of a run see different pages, a page whose V scale is 2^r times the others' leaves the rows
    // that do not see it probabilities off by 2^(r - 31) of the largest: as much as an fp16 output's rounding at r = 20. A
    // reference per column costs 82.7 -> 101.2 us at 24 x 8 tokens behind 8000 and up to 5 % for single tokens, whose
    // columns all see the same.
    float vref = 0.0f, vmul = 0.0f;
    const float second = FOLD && t >= 2 ? 1.0f : 0.0f;

    // Scores of TP tiles -> probabilities as B fragments pb; also the running state. Whether all rows see all of them.
    auto softmax = [&](auto tp, float (*s)[NT][4], const float* f, const float* vs, const int* key0, int item, int live,
                       uint32_t (*pb)[NT][4]) {
        constexpr int TP = decltype(tp)::value;
        bool whole = true, raise = false;
        float vtop = vs[0];
#pragma unroll
        for (int i = 0; i < TP; ++i) whole = whole && key0[i] + 15 <= v.pos0 && (key0[i] >= v.low1 || key0[i] + 16 <= p.sinks);
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][nt][e] *= f[i];
        if (!whole) {
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0[i] + g + (e >> 1) * 8, c = e & 1;
                        if (key > hi[nt][c] || (key < lo[nt][c] && key >= p.sinks)) s[i][nt][e] = -INFINITY;
                    }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                for (int i = 1; i < TP; ++i) top = fmaxf(top, fmaxf(s[i][nt][c], s[i][nt][c + 2]));
                raise |= top > m[nt][c] + kQ8Lazy;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                    for (int i = 1; i < TP; ++i) top = fmaxf(top, fmaxf(s[i][nt][c], s[i][nt][c + 2]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float mn = fmaxf(m[nt][c], top), a = fast_exp2(m[nt][c] - mn);
                    m[nt][c] = mn;
                    l[nt][c] *= a;
#pragma unroll
                    for (int mt = 0; mt < T::MT; ++mt) { o[nt][mt][c] *= a; o[nt][mt][c + 2] *= a; }
                }
        }
#pragma unroll
        for (int i = 1; i < TP; ++i) vtop = fmaxf(vtop, vs[i]);
        if (vtop > vref) {   // uniform over the warp; NaN scales do not count and go through as they are
            const float next = __uint_as_float((__float_as_uint(vtop) & 0x7f800000u) + 0x00800000u), a = vref / next;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < T::MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][mt][e] *= a;
            vref = next;
            vmul = kQ8Headroom / next;
        }
#pragma unroll
        for (int i = 0; i < TP; ++i) {
            const float w = vs[i] * vmul;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = fast_exp2(s[i][nt][k] - m[nt][k & 1]);
                l[nt][0] += e[0] + e[2];
                l[nt][1] += e[1] + e[3];
                if constexpr (MASS) {
                    // sums over the 16 tokens: lanes of even g end up with column 2t's, those of odd g with column 2t + 1's
                    const bool odd = g & 1;
                    const float a = e[0] + e[2], b = e[1] + e[3];
                    float x = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    // a column that holds no row leaves 0, whatever 0 times an infinite key made of it
                    if (g < 2 && i < live)
                        p.page_ws[((size_t)(seq * nkv + h) * p.ws_tiles + item + i) * R + 8 * nt + 2 * t + g] =
                            make_float2((g ? hi[nt][1] : hi[nt][0]) < 0 ? 0.0f : x, g ? m[nt][1] : m[nt][0]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // a probability of a masked key is 0 whatever the page's scale is
                    if (!whole && s[i][nt][k] == -INFINITY) e[k] = 0.0f;
                    else e[k] *= w;
                }
                const uint32_t h0 = pack_half2(e[0], e[1]), h1 = pack_half2(e[2], e[3]);
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                if (FOLD) {   // columns 4 .. 7 have the probabilities of 0 .. 3 and take what fp16 leaves of them
                    pb[i][nt][0] = movmatrix_trans(pack_half2(fmaf(-second, f0.x, e[0]), fmaf(-second, f0.y, e[1])));
                    pb[i][nt][1] = movmatrix_trans(pack_half2(fmaf(-second, f1.x, e[2]), fmaf(-second, f1.y, e[3])));
                } else {
                    pb[i][nt][0] = movmatrix_trans(h0);
                    pb[i][nt][1] = movmatrix_trans(h1);
                    pb[i][nt][2] = movmatrix_trans(pack_half2(e[0] - f0.x, e[1] - f0.y));
                    pb[i][nt][3] = movmatrix_trans(pack_half2(e[2] - f1.x, e[3] - f1.y));
                }
            }
        }
        return whole;
    };
    // Whether a token of a partly visible tile is seen by no row of this block.
    auto unseen = [&](int key) { return key >= v.end || (key < v.low0 && key >= p.sinks); };

    // ---- page tiles: a ring of S stages per warp, filled by the lanes for themselves
    const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * S * TPI) * T::STAGE;
    const int q1 = min(i1, v.tiles);
    const int* table = p.seq.tables + (size_t)seq * p.seq.width;
    const int sub_mask = (block >> 4) - 1, sub_log = p.cache.log2b - 4;
    auto tile_of = [&](int item) { return item < v.ns ? item : item - v.ns + v.w0; };
    // A warp takes TPI neighbouring tiles at a time. Tile `a` of a warp, and the item a copy that is due reads: the last of
    // an odd number is copied twice and masked, so that no stage ever holds anything but codes.
    auto item_of = [&](int a) {
        const int item = i0 + TPI * (warp + a / TPI * kWarps) + a % TPI;
        return TPI > 1 && a % TPI && item == q1 ? item - 1 : item;
    };
    // Page ids of the warp's tiles, 32 at a time, one per lane, a block of 32 ahead of their use: the load's latency and
    // the check against the pool are paid once per 32 tiles.
    auto load_ids = [&](int a0) {
        const int item = item_of(a0 + lane);
        const int page = item < q1 ? tile_of(item) >> sub_log : 0;
        return item < q1 && page < p.seq.width ? table[page] : item < q1 ? -1 : 0;
    };
    auto checked = [&](int id) {
        if (!index_in_pool(id, p.cache.num_blocks)) { atomicAdd(&g_q8_attn_rejected, 1u); id = 0; }
        return id;
    };
    const size_t page_bytes = (size_t)nkv * block * D;
    const uint8_t* kbase = p.cache.k + (size_t)h * block * D + lane * 16;
    const uint8_t* vbase = p.cache.v + (size_t)h * block * D + lane * 16;
    // chunk 32 i + lane of a tile: row (32 i + lane) / CPR; rows of later i are a multiple of 2 on (of 8 at D = 64, where
    // the swizzle depends on three bits of the row; of 4 and 2 at D = 128 and 256)
    auto swizzled = [&](int i, bool is_v) {
        const int row = (32 * i + lane) / T::CPR, chunk = lane % T::CPR;
        return (uint32_t)(row * D + ((chunk ^ (is_v ? T::v_swizzle(row) : T::k_swizzle(row))) << 4));
    };
    auto issue = [&](int item, int id, uint32_t dst) {
        if (item < q1) {
            const size_t at = (size_t)id * page_bytes + (size_t)(tile_of(item) & sub_mask) * T::BYTES;
            const uint8_t *k = kbase + at, *vv = vbase + at;
#pragma unroll
            for (int i = 0; i < T::BYTES / 512; ++i) cp_async16_32(dst + swizzled(i, false), k + 512 * i);
#pragma unroll
            for (int i = 0; i < T::BYTES / 512; ++i) cp_async16_32(dst + T::BYTES + swizzled(i, true), vv + 512 * i);
            if (lane == 0) cp_async8(dst + 2 * T::BYTES, p.cache.scales + (size_t)id * nkv + h);
        }
    };
    // where this lane's pieces lie in a stage
    const uint32_t k_at = g * D + ((t ^ T::k_swizzle(g)) << 4);
    const uint32_t v_at = T::BYTES + 2 * t * D + (D == 64 ? (((g >> 1) ^ T::v_swizzle(2 * t)) << 4) + (g & 1) * 8 : (g ^ T::v_swizzle(2 * t)) << 4);
    {
        int ids = checked(load_ids(0)), ids_next = load_ids(32), asked = 0;
        auto issue_next = [&](int stage) {
#pragma unroll
            for (int i = 0; i < TPI; ++i) {
                const int id = __shfl_sync(0xffffffffu, ids, (asked + i) & 31);
                issue(item_of(asked + i), id, ring + (uint32_t)(stage * TPI + i) * T::STAGE);
            }
            cp_async_commit();
            asked += TPI;
            if ((asked & 31) == 0) { ids = checked(ids_next); ids_next = load_ids(asked + 32); }
        };
#pragma unroll
        for (int s = 0; s < S - 1; ++s) issue_next(s);
        int stage = 0;
        for (int item = i0 + TPI * warp; item < q1; item += TPI * kWarps) {
            issue_next(stage == 0 ? S - 1 : stage - 1);
            cp_async_wait<S - 1>();
            __syncwarp();                          // the other lanes' copies have landed too
            const uint32_t src = ring + (uint32_t)(stage * TPI) * T::STAGE;
            const int live = TPI > 1 && item + 1 == q1 ? 1 : TPI;
            float s[TPI][NT][4], f[TPI], vs[TPI];
            int key0[TPI];
            uint32_t pb[TPI][NT][4];
#pragma unroll
            for (int tt = 0; tt < TPI; ++tt) {
                const uint2 sc = lds64(src + tt * T::STAGE + 2 * T::BYTES);
                f[tt] = __uint_as_float(sc.x) * p.scale_log2;
                vs[tt] = __uint_as_float(sc.y);
                key0[tt] = tt < live ? tile_of(item + tt) * 16 : 0x3fffffff;   // no row sees that far
                float s2[NT][4];   // two sums, so that half as many products wait on one another
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[tt][nt][e] = s2[nt][e] = 0.0f;
#pragma unroll
                for (int j = 0; j < T::KC; ++j) {
                    // piece t + 4 j: the swizzle flips bit 2 of the chunk, that is j's low bit
                    const uint32_t at = src + tt * T::STAGE + (k_at ^ (uint32_t)((j & 1) << 6)) + (j >> 1) * 128;
                    const uint4 a = lds128(at), b = lds128(at + 8 * D);
                    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        q8_unpack<FMT>(aw[i], a0, a2);
                        q8_unpack<FMT>(bw[i], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            product(i & 1 ? s2[nt] : s[tt][nt], a0, a1, a2, a3, qf[nt][4 * j + i][0], qf[nt][4 * j + i][1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[tt][nt][e] += s2[nt][e];
            }
            const bool whole = softmax(std::integral_constant<int, TPI>(), s, f, vs, key0, item, live, pb);
#pragma unroll
            for (int tt = 0; tt < TPI; ++tt)
#pragma unroll
                for (int j = 0; j < T::VP; ++j) {
                    uint32_t w[4][T::VW];
                    const uint32_t at = src + tt * T::STAGE + v_at + j * 128;
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const int row = (k4 & 1) + (k4 >> 1) * 8;
                        if constexpr (T::VB == 8) {
                            const uint2 x = lds64(at + row * D);
                            w[k4][0] = x.x; w[k4][1] = x.y;
                        } else {
                            const uint4 x = lds128(at + row * D);
                            w[k4][0] = x.x; w[k4][1] = x.y; w[k4][2] = x.z; w[k4][3] = x.w;
                        }
                        if (!whole && unseen(key0[tt] + 2 * t + row)) {
#pragma unroll
                            for (int i = 0; i < T::VW; ++i) w[k4][i] = 0u;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < T::VW; ++i) {
                        uint32_t ab[4], cd[4];
                        q8_unpack_pairs<FMT>(w[0][i], w[1][i], ab);
                        q8_unpack_pairs<FMT>(w[2][i], w[3][i], cd);
                        const int mt = 8 * j + 2 * i;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            product(o[nt][mt], ab[0], ab[1], cd[0], cd[1], pb[tt][nt][0], pb[tt][nt][1]);
                            product(o[nt][mt + 1], ab[2], ab[3], cd[2], cd[3], pb[tt][nt][0], pb[tt][nt][1]);
                            if (!FOLD) {
                                product(o[nt][mt], ab[0], ab[1], cd[0], cd[1], pb[tt][nt][2], pb[tt][nt][3]);
                                product(o[nt][mt + 1], ab[2], ab[3], cd[2], cd[3], pb[tt][nt][2], pb[tt][nt][3]);
                            }
                        }
                    }
                }
            stage = stage == S - 1 ? 0 : stage + 1;
            __syncwarp();                          // every lane has read the stage that the next copies go to
        }
    }

    // ---- tail tiles: fp16 rows straight from global memory (at most B / 16 of them per sequence)
    if (i1 > v.tiles) {
        int slot = q8_slot(p.seq, seq);
        if (!index_in_pool(slot, p.cache.num_slots)) {
            if (lane == 0 && warp == 0) atomicAdd(&g_q8_attn_rejected, 1u);
            slot = 0;
        }
        const __half* kt = p.cache.k_tail + ((size_t)slot * nkv + h) * block * D;
        const __half* vt = p.cache.v_tail + ((size_t)slot * nkv + h) * block * D;
        for (int item = max(i0, v.tiles) + warp; item < i1; item += kWarps) {
            const int r0 = (item - v.tiles) * 16, key0 = v.paged + r0;
            auto word4 = [&](const __half* base, int row, int chan) {   // 8 channels of a token, zero unless it is seen
                if (unseen(v.paged + row)) return make_uint4(0u, 0u, 0u, 0u);
                return *reinterpret_cast<const uint4*>(base + (size_t)row * D + chan);
            };
            float s[1][NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[0][nt][0] = s[0][nt][1] = s[0][nt][2] = s[0][nt][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < T::KC; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 a = word4(kt, r0 + g, 16 * t + 64 * j + 8 * half), b = word4(kt, r0 + g + 8, 16 * t + 64 * j + 8 * half);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        product(s[0][nt], a.x, b.x, a.y, b.y, qf[nt][4 * j + 2 * half][0], qf[nt][4 * j + 2 * half][1]);
                        product(s[0][nt], a.z, b.z, a.w, b.w, qf[nt][4 * j + 2 * half + 1][0], qf[nt][4 * j + 2 * half + 1][1]);
                    }
                }
            uint32_t pb[1][NT][4];
            const float unit_scale = 1.0f;
            softmax(std::integral_constant<int, 1>(), s, &p.scale_log2, &unit_scale, &key0, item, 1, pb);
            uint32_t seen = 0;                      // bit 4 nt + e: whether score e's row sees its key
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) seen |= (s[0][nt][e] != -INFINITY ? 1u : 0u) << (4 * nt + e);
            auto ones = [&](int bit) { return movmatrix_trans((seen >> bit & 1u) * 0x3c00u + (seen >> (bit + 1) & 1u) * 0x3c000000u); };
#pragma unroll
            for (int e = 0; e < T::MT / 4; ++e) {   // 8 channels of a token per 16-byte word: output tiles 4 e .. 4 e + 3
                const int chan = D == 64 ? 8 * g : 16 * g + 8 * (e & 1) + 128 * (e >> 1);
                uint4 x[4];
                bool odd = false;
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                    x[k4] = word4(vt, r0 + 2 * t + (k4 & 1) + (k4 >> 1) * 8, chan);
                    const uint32_t w[4] = {x[k4].x, x[k4].y, x[k4].z, x[k4].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd |= (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
                }
                uint32_t a[4][4];                   // [tile][fragment register]
                auto pairs = [&](const uint4& y0, const uint4& y1, int reg) {
                    const uint32_t w0[4] = {y0.x, y0.y, y0.z, y0.w}, w1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[i][reg] = __byte_perm(w0[i], w1[i], 0x5410);
                        a[i][reg + 1] = __byte_perm(w0[i], w1[i], 0x7632);
                    }
                };
                pairs(x[0], x[1], 0);
                pairs(x[2], x[3], 2);
                // An infinity or NaN in V must reach the rows that see its token and no other, but 0 * NaN is NaN: such
                // elements leave the product, and a second product counts those that a row sees (not their weight, which may
                // have underflowed).
                const bool any_odd = __any_sync(0xffffffffu, odd);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t bad[4] = {0u, 0u, 0u, 0u};
                    if (any_odd) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if ((a[i][k] & 0x7c00u) == 0x7c00u) { a[i][k] &= 0xffff0000u; bad[k] |= 0x3c00u; }
                            if ((a[i][k] & 0x7c000000u) == 0x7c000000u) { a[i][k] &= 0x0000ffffu; bad[k] |= 0x3c000000u; }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        product(o[nt][4 * e + i], a[i][0], a[i][1], a[i][2], a[i][3], pb[0][nt][0], pb[0][nt][1]);
                        if (!FOLD) product(o[nt][4 * e + i], a[i][0], a[i][1], a[i][2], a[i][3], pb[0][nt][2], pb[0][nt][3]);
                        if (any_odd) {
                            float hit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            product(hit, bad[0], bad[1], bad[2], bad[3], ones(4 * nt), ones(4 * nt + 2));
#pragma unroll
                            for (int k = 0; k < 4; ++k) if (hit[k] != 0.0f) o[nt][4 * e + i][k] = __int_as_float(0x7fc00000);
                        }
                    }
                }
            }
        }
    }

    // ---- merge: the CTA's warps through shared memory (over the ring), then the cluster's CTAs
    cp_async_wait<0>();
    const float back = vref / kQ8Headroom;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float x = l[nt][c];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            if (g == 0) { s_m[warp][8 * nt + 2 * t + c] = m[nt][c]; s_l[warp][8 * nt + 2 * t + c] = x; }
        }
    __syncthreads();                              // rings are drained, states are there
    // Accumulators lie in fragment order, [warp][accumulator][lane]: neighbouring lanes in neighbouring banks.
    constexpr int ACC = NT * T::MT * 4, VEC = ACC * 32;
    float* so = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = 8 * nt + 2 * t + c;
            float top = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
            const float a = back * fast_exp2(m[nt][c] - top);
#pragma unroll
            for (int mt = 0; mt < T::MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    so[warp * VEC + ((nt * T::MT + mt) * 4 + 2 * hf + c) * 32 + lane] = o[nt][mt][2 * hf + c] * a;
        }
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float top = s_m[0][r], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s_l[w][r] * fast_exp2(s_m[w][r] - top);
        c_m[r] = top; c_l[r] = sum;
    }
    __syncthreads();
    constexpr int QUADS = T::MT / 4, ITEMS = NT * 2 * QUADS * 32;
    if (p.parts > 1 && p.cluster == 0) {         // partials for the merge kernel, row by row
        pdl_trigger();
        const size_t slot = (size_t)unit * p.parts + part;
        for (int e = threadIdx.x; e < R * D / 4; e += kWarps * 32) {
            const int r = e / (D / 4), at = accumulator_of<D>(r, e % (D / 4) * 4);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)   // channel + 1: two accumulators further; column + 4: two lanes
                    x[k] += so[w * VEC + at + k * 64] + (FOLD && r < 4 ? so[w * VEC + at + k * 64 + 2] : 0.0f);
            reinterpret_cast<float4*>(p.part_o)[slot * (R * D / 4) + e] = make_float4(x[0], x[1], x[2], x[3]);
        }
        if (threadIdx.x < R) p.part_ml[slot * R + threadIdx.x] = make_float2(c_m[threadIdx.x], c_l[threadIdx.x]);
        return;
    }
    if (p.parts > 1) {
        for (int e = threadIdx.x; e < VEC; e += kWarps * 32) {
            float x = so[e];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) x += so[w * VEC + e];
            so[e] = x;
        }
        cg::this_cluster().sync();
    }
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float top = c_m[r], sum = c_l[r];
        if (p.parts > 1) {
            auto cluster = cg::this_cluster();
            for (int c = 0; c < p.parts; ++c) top = fmaxf(top, *cluster.map_shared_rank(&c_m[r], c));
            sum = 0.0f;
            for (int c = 0; c < p.parts; ++c)
                sum += *cluster.map_shared_rank(&c_l[r], c) * fast_exp2(*cluster.map_shared_rank(&c_m[r], c) - top);
        }
        f_m[r] = top;
        // a row that saw nothing has sum 0 and o 0; rows behind the block's last weigh nothing
        f_il[r] = sum != 0.0f && rb * R + r < rows ? 1.0f / sum : 0.0f;
    }
    __syncthreads();
    // An item: 8 consecutive channels (4 accumulator tiles) of one row, in one lane's place; shared out over the cluster.
    const int share = (ITEMS + p.parts - 1) / p.parts;
    for (int e = part * share + threadIdx.x; e < min(ITEMS, (part + 1) * share); e += kWarps * 32) {
        const int el = e & 31, q4 = (e >> 5) % QUADS, c = (e >> 5) / QUADS & 1, nt = (e >> 5) / QUADS >> 1;
        const int r = 8 * nt + 2 * (el & 3) + c, row = rb * R + r;
        if (row >= rows) continue;
        float x[8];
        const float* src = so + ((nt * T::MT + 4 * q4) * 4 + c) * 32 + el;   // channel 2 i + hf: 4 i + 2 hf accumulators further
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = 0.0f;
        if (p.parts > 1) {
            auto cluster = cg::this_cluster();
            for (int rank = 0; rank < p.parts; ++rank) {
                const float a = fast_exp2(*cluster.map_shared_rank(&c_m[r], rank) - f_m[r]);
                const float* peer = cluster.map_shared_rank(src, rank);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] += a * (peer[k * 64] + (FOLD ? peer[k * 64 + 2] : 0.0f));
            }
        } else {
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] += src[w * VEC + k * 64] + (FOLD ? src[w * VEC + k * 64 + 2] : 0.0f);
        }
        const float il = f_il[r];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= il;
        store8(p, out_at(p, u, row, D) + channel_of<D>(el >> 2, 4 * q4, 0), x);
    }
    if constexpr (MASS) add_masses<R>(p, u, f_m, f_il, part * kWarps * 32 + threadIdx.x, p.parts * kWarps * 32);
    if (p.parts > 1) cg::this_cluster().sync();   // nobody leaves while a peer may still read its shared memory
}

// Joins the parts of a unit that was cut without a cluster. grid (units, slices): slice 0 writes the output, all share
// the pages' masses out. Launched early (programmatic dependent launch): what it reads of the caller's is not written by
// the kernel before it, and of that kernel's results it reads nothing before the wait.
template <int D, int NT, bool MASS>
__global__ void __launch_bounds__(256) q8_merge_kernel(const Q8AttnParams p) {
    constexpr int R = 8 * NT;
    __shared__ float f_m[R], f_il[R], weight[kMaxParts][R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Unit u = make_unit(p, blockIdx.x, R);
    const int live = max(1, (u.items + p.chunk - 1) / p.chunk);
    pdl_wait();
    if (u.rb * R >= u.rows) return;
    const float2* ml = p.part_ml + (size_t)blockIdx.x * p.parts * R;
    for (int r = warp; r < R; r += 8) {          // a lane per part
        const float2 x = lane < live ? ml[lane * R + r] : make_float2(kQ8Unset, 0.0f);
        float top = x.x;
#pragma unroll
        for (int k = 16; k > 0; k /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float a = fast_exp2(x.x - top);
        float sum = x.y * a;
#pragma unroll
        for (int k = 16; k > 0; k /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        const float il = sum != 0.0f && u.rb * R + r < u.rows ? 1.0f / sum : 0.0f;
        weight[lane][r] = a * il;
        if (lane == 0) { f_m[r] = top; f_il[r] = il; }
    }
    __syncthreads();
    if (blockIdx.y == 0) {
        for (int e = threadIdx.x; e < R * D / 4; e += 256) {
            const int r = e / (D / 4), row = u.rb * R + r;
            if (row >= u.rows) continue;
            const float4* src = reinterpret_cast<const float4*>(p.part_o) + (size_t)blockIdx.x * p.parts * (R * D / 4) + e;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
            for (int part = 0; part < live; ++part) {
                const float4 y = __ldcg(src + (size_t)part * (R * D / 4));
                const float a = weight[part][r];
                x.x += a * y.x; x.y += a * y.y; x.z += a * y.z; x.w += a * y.w;
            }
            const size_t at = out_at(p, u, row, D) + e % (D / 4) * 4;
            if (p.out_h) *reinterpret_cast<uint2*>(p.out_h + at) = make_uint2(pack_half2(x.x, x.y), pack_half2(x.z, x.w));
            else *reinterpret_cast<float4*>(p.out + at) = x;
        }
    }
    if constexpr (MASS) add_masses<R>(p, u, f_m, f_il, blockIdx.y * 256 + threadIdx.x, gridDim.y * 256);
}

template <int D, int FMT, int ROWS, bool MASS, int kWarps>
cudaError_t launch(const Q8AttnParams& p, cudaStream_t stream) {
    constexpr int NT = ROWS == kRows16 ? 2 : 1;
    constexpr size_t ring = (size_t)kWarps * stages_of<D, kWarps>() * tiles_at_once(D) * Tile<D>::STAGE, merge = (size_t)kWarps * 8 * NT * D * 4;
    constexpr size_t smem = ring > merge ? ring : merge;
    auto kernel = q8_attention_kernel<D, FMT, ROWS, MASS, kWarps, NT>;
    static Q8SmemLimit limit;
    cudaError_t e = limit.raise(kernel, (int)smem);
    if (e != cudaSuccess) return e;
    const unsigned units = (unsigned)((size_t)p.seq.batch * p.cache.nkv * p.row_blocks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units * p.parts);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess || p.parts == 1 || p.cluster) return e;
    const unsigned slices = MASS ? (unsigned)((((p.max_seq >> p.cache.log2b) + 1) + 511) / 512) : 1u;
    cudaLaunchConfig_t merge_cfg = {};
    merge_cfg.gridDim = dim3(units, slices < 64 ? slices : 64);
    merge_cfg.blockDim = dim3(256);
    merge_cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    merge_cfg.attrs = attr;
    merge_cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&merge_cfg, q8_merge_kernel<D, NT, MASS>, p);
}

template <int D, int FMT, bool MASS, int kWarps>
cudaError_t launch_shape(const Q8AttnParams& p, int rows, cudaStream_t stream) {
    return rows == kRows4 ? launch<D, FMT, kRows4, MASS, kWarps>(p, stream)
         : rows == kRows8 ? launch<D, FMT, kRows8, MASS, kWarps>(p, stream) : launch<D, FMT, kRows16, MASS, kWarps>(p, stream);
}

template <int D, int FMT>
cudaError_t launch_rows(Q8AttnParams p, int warps, cudaStream_t stream) {
    const int n = p.max_q * p.qpk, r = n > 8 ? 16 : 8, blocks = (n + r - 1) / r;
    const int rows = n <= 4 ? kRows4 : n <= 8 ? kRows8 : kRows16;
    if (!p.mass) {
        p.row_blocks = blocks; p.row_block0 = 0;
        return warps == 4 ? launch_shape<D, FMT, false, 4>(p, rows, stream) : launch_shape<D, FMT, false, 8>(p, rows, stream);
    }
    // page masses of a kv head grow by one block of query heads at a time: its own launch, so nothing races
    p.row_blocks = 1;
    for (p.row_block0 = 0; p.row_block0 < blocks; ++p.row_block0) {
        const cudaError_t e = warps == 4 ? launch_shape<D, FMT, true, 4>(p, rows, stream) : launch_shape<D, FMT, true, 8>(p, rows, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Tiles of the longest unit the launch allows: the window of a block of rows, the first tokens, what the two share of
// tiles at their ends, and the tail, all of whose tiles are visited. Exceeding it would cut units short: View counts the
// same way.
int most_tiles(int max_q, int max_seq, int window, int sinks, int block) {
    const long long whole = max_seq, part = (long long)window + max_q + sinks + block + 48;
    return (int)(((window != 0x7fffffff && part < whole ? part : whole) + 15) / 16) + 2;
}

struct Plan {
    bool wide;                 // 16 query rows per unit, else 8
    bool prompt;               // the kernel for many rows
    int tiles, units;          // of the longest unit; units of a launch
    int parts, chunk, cluster, warps;
    size_t page_ws, part_ml, part_o, total;   // workspace: offsets and size
};

// How many parts a unit's context is cut into, and whether the parts form a cluster. The model, in us, fitted to
// measurements at 8192 and 32768 tokens: a CTA costs kStart before and after its tiles; a warp's two tiles (one at
// D = 256) take pair_us[c - 1] with c CTAs on a multiprocessor (the copy rate bounds it from c = 2 on at D = 128); a
// multiprocessor runs its queue in rounds of as many CTAs as fit. Parts are joined in a cluster (about 1 us, parts 2, 4
// or 8) while all clusters are resident at once -- 16 units of 512 tokens, head_dim 64: 6.8 us against 8.2 with the
// merge kernel -- and by the merge kernel beyond that (256 units of ragged lengths in 2 parts: 63 us against 56, as
// clusters wait for all of their CTAs' slots). All sequences are cut by the longest one's tiles: in a ragged batch the
// longest sequence's parts decide the time while others' places are empty. The figures here are all the model was fitted
// to; it was not measured on a second set of calls. With one unit per multiprocessor or fewer, eight-warp CTAs with deeper
// rings (8 units of 32768 tokens: 24.7 us against 26.6).
constexpr double kStart = 4.0, kClusterUs = 1.0, kMergeUs = 3.0;
constexpr long long kMostParts = 16384;

void plan_parts(Plan& q, int d) {
    static const double pair64[4] = {0.95, 1.16, 1.42, 1.73}, pair128[3] = {1.08, 1.57, 2.45}, pair256[2] = {1.3, 2.4};
    const double* pair_us = d == 64 ? pair64 : d == 128 ? pair128 : pair256;
    const int resident = d == 64 ? 4 : d == 128 ? 3 : 2, sms = sm_count(), at_once = tiles_at_once(d);
    const double slow = q.wide ? 1.25 : 1.0;
    double best = 1e30;
    auto chunk_of = [&](int parts) { return ((q.tiles + parts - 1) / parts + 1) / 2 * 2; };
    auto offer = [&](int parts, int cluster, int warps) {
        const long long queue = ((long long)q.units * parts + sms - 1) / sms;
        const int pairs = (chunk_of(parts) + warps * at_once - 1) / (warps * at_once);
        double t = parts == 1 ? 0.0 : cluster ? kClusterUs : kMergeUs;
        if (warps == 8) {
            t += (double)queue * (kStart + pairs * slow * pair_us[1]);
        } else {
            const int rest = (int)(queue % resident);
            t += (double)(queue / resident) * (kStart + pairs * slow * pair_us[resident - 1]);
            if (rest) t += kStart + pairs * slow * pair_us[rest - 1];
        }
        // lengths of a batch differ, and a launch of whole units is as long as its longest: 256 units of 500 .. 6000 tokens
        // take 69 us whole and 56 in two parts, 1024 equal ones of 8192 tokens 356 and 349
        t *= parts > 1 ? 1.03 : q.tiles >= 192 && q.units > 1 ? 1.15 : 1.0;
        if (t < best) { best = t; q.parts = parts; q.cluster = cluster; q.warps = warps; }
    };
    offer(1, 0, 4);
    // partials cost 8 D bytes a row and part: beyond this many parts the launch is even enough without
    for (int parts = 2; parts <= kMaxParts && q.tiles >= parts * 4 && (long long)q.units * parts <= kMostParts; ++parts) {
        const bool fits = (long long)q.units * parts <= (long long)resident * sms;
        if (fits && (parts == 2 || parts == 4 || parts == 8)) offer(parts, 1, 4);
        else offer(parts, 0, 4);
        if ((long long)q.units * parts <= sms && q.tiles >= parts * 32) offer(parts, 0, 8);
    }
    q.chunk = chunk_of(q.parts);
}

// Whether the kernel for many rows is the faster one. It takes 3.1, 3.8 and 4.6 us (head_dim 64, 128, 256) for 128 keys of
// its 256 (128) rows on every multiprocessor; the other one 0.40, 0.60 and 1.3 ns for 16 keys of 16 rows. At head_dim
// 128, 8 sequences of 8192 tokens, 8 kv heads: 128 rows each 272 us against 192, 256 rows 280 against 482, 512 rows
// 281 against 934. Over two sets of 36 calls between both kernels' ranges it takes 1.0 and 2.0 % more than the faster
// kernel of each call, always the one for few rows 15 and 11 %, always the other 29 and 25 % (geometric means). It loses 3
// to 8 us on small calls (128, 4 x 104 tokens, 2/14 heads: 15.8 -> 23.3), and misses one large one: 64, 3 x 150 tokens
// behind 5163, 3/36 heads, 180 us against 139. It knows the largest count of the batch only: single tokens beside a prompt
// go with the prompt, in units of 256 rows of which they fill a few; a caller that has many makes two calls.
bool many_rows(int d, int batch, int nkv, long long rows, int tiles) {
    const int per = d == 256 ? 128 : 256;
    const double step_us = d == 64 ? 3.1 : d == 128 ? 3.8 : 4.6, tile_us = (d == 64 ? 0.40 : d == 128 ? 0.60 : 1.3) * 1e-3;
    const long long units = (long long)batch * nkv * ((rows + per - 1) / per), rounds = (units + sm_count() - 1) / sm_count();
    const double many = 15.0 + (double)rounds * ((tiles + 7) / 8) * step_us;
    const double few = 20.0 + (double)batch * nkv * ((rows + 15) / 16) * tiles * tile_us;
    return rows > 16 && 1.1 * many < few;
}

Plan make_plan(int nkv, int qpk, int d, int block, int batch, int max_q, int max_seq, int window, int sinks, bool mass) {
    Plan q = {};
    const long long rows = (long long)max_q * qpk;
    q.wide = rows > 8;
    const int r = q.wide ? 16 : 8;
    q.tiles = most_tiles(max_q, max_seq, window, sinks, block);
    q.prompt = !mass && many_rows(d, batch, nkv, rows, q.tiles);
    if (q.prompt) return q;
    q.units = (int)((long long)batch * nkv * (mass ? 1 : (rows + r - 1) / r));
    plan_parts(q, d);
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    size_t at = 0;
    q.page_ws = at;
    if (mass) at += up((size_t)batch * nkv * q.tiles * r * sizeof(float2));
    if (q.parts > 1 && !q.cluster) {
        q.part_ml = at; at += up((size_t)q.units * q.parts * r * sizeof(float2));
        q.part_o = at; at += up((size_t)q.units * q.parts * r * d * sizeof(float));
    }
    q.total = at;
    return q;
}

}  // namespace

size_t q8_attention_workspace(int nkv, int qpk, int d, int block, int batch, int max_q, int max_seq, int window, int sinks, bool mass) {
    return make_plan(nkv, qpk, d, block, batch, max_q, max_seq, window, sinks, mass).total;
}

cudaError_t launch_q8_attention(const Q8AttnParams& args, int d, int fmt, void* workspace, cudaStream_t stream) {
    Q8AttnParams p = args;
    const Plan plan = make_plan(p.cache.nkv, p.qpk, d, 1 << p.cache.log2b, p.seq.batch, p.max_q, p.max_seq, p.window, p.sinks, p.mass != nullptr);
    if (plan.prompt) return launch_q8_prompt(p, d, fmt, stream);
    p.ws_tiles = plan.tiles;
    p.parts = plan.parts; p.chunk = plan.chunk; p.cluster = plan.cluster;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    p.page_ws = reinterpret_cast<float2*>(ws + plan.page_ws);
    p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
    p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
    const bool i8 = fmt == KIVI_Q8_INT8;
    const int warps = plan.warps;
    switch (d) {
        case 64: return i8 ? launch_rows<64, KIVI_Q8_INT8>(p, warps, stream) : launch_rows<64, KIVI_Q8_E4M3>(p, warps, stream);
        case 128: return i8 ? launch_rows<128, KIVI_Q8_INT8>(p, warps, stream) : launch_rows<128, KIVI_Q8_E4M3>(p, warps, stream);
        default: return i8 ? launch_rows<256, KIVI_Q8_INT8>(p, warps, stream) : launch_rows<256, KIVI_Q8_E4M3>(p, warps, stream);
    }
}

cudaError_t q8_attention_rejected(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_q8_attn_rejected, sizeof(*count)); }

}  // namespace kivi
