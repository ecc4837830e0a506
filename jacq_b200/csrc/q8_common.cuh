// Shared by the kernels of the 8-bit block-scaled cache: its pointers, how a launch finds a sequence, conversions.
#pragma once

#include <atomic>

#include "kivi_common.cuh"

namespace kivi {

constexpr float kQ8RecipInt8 = 1.0f / 127.0f;
constexpr float kQ8RecipE4m3 = 1.0f / 448.0f;

struct Q8Cache {
    uint8_t* k; uint8_t* v;        // [num_blocks, NKV, B, D] codes
    float2* scales;                // [num_blocks, NKV] (K, V)
    __half* k_tail; __half* v_tail;  // [num_slots, NKV, B, D]
    int num_blocks, num_slots;
    int nkv, log2b;
};

struct Q8Seqs {
    const int* tables; int width;  // [batch, width]
    const int* lens;               // [batch]
    const int* slots;              // [batch] or nullptr: slot i
    int batch;
};

__device__ __forceinline__ int q8_slot(const Q8Seqs& s, int i) { return s.slots ? s.slots[i] : i; }

// Sequences and ids a launch refused (kivi_b200_q8_rejected_indices adds the files' counters up).
cudaError_t q8_cache_rejected(unsigned int* count);
cudaError_t q8_attention_rejected(unsigned int* count);
cudaError_t q8_prompt_rejected(unsigned int* count);
cudaError_t q8_evict_rejected(unsigned int* count);

// Two codes (the low 16 bits of `codes`) as a pair of fp16 values; every e4m3 value is an fp16 value.
__device__ __forceinline__ uint32_t q8_e4m3_pair(uint16_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
    return r;
}
// Two int8 codes that were biased to 1024 + 128 + code by a byte permute under 0x64: minus 1152 is exact.
__device__ __forceinline__ uint32_t q8_int8_pair(uint32_t biased) {
    const __half2 bias = __halves2half2(__ushort_as_half((unsigned short)0xE480), __ushort_as_half((unsigned short)0xE480));
    const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&biased), bias);
    return *reinterpret_cast<const uint32_t*>(&x);
}

// Codes c0 c1 c2 c3 of one word as the pairs (c0, c1) and (c2, c3).
template <int FMT>
__device__ __forceinline__ void q8_unpack(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == KIVI_Q8_INT8) {
        w ^= 0x80808080u;
        lo = q8_int8_pair(__byte_perm(w, 0x64646464u, 0x4140));
        hi = q8_int8_pair(__byte_perm(w, 0x64646464u, 0x4342));
    } else {
        lo = q8_e4m3_pair((uint16_t)w);
        hi = q8_e4m3_pair((uint16_t)(w >> 16));
    }
}

// Words a and b of two tokens, the same four channels: pairs (a_c, b_c) for c = 0 .. 3.
template <int FMT>
__device__ __forceinline__ void q8_unpack_pairs(uint32_t a, uint32_t b, uint32_t (&p)[4]) {
    const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
    q8_unpack<FMT>(x, p[0], p[1]);
    q8_unpack<FMT>(y, p[2], p[3]);
}

// A kernel's dynamic shared memory limit, raised once per device (a microsecond of every launch otherwise).
struct Q8SmemLimit {
    std::atomic<bool> done[64] = {};
    template <class Kernel>
    cudaError_t raise(Kernel kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
        return e;
    }
};

// Host launchers.
struct Q8WriteParams {
    Q8Cache cache; Q8Seqs seq;     // seq.lens: tokens before the call
    const __half* new_k; const __half* new_v;
    long long k_stride, v_stride;
    const int* offsets;
    int total_new, max_new, max_start;
};
struct Q8ReadParams {
    Q8Cache cache; Q8Seqs seq;
    const int* offsets; const int* first;
    int total_rows, max_rows;
    __half* k_out; __half* v_out;
};
struct Q8AttnParams {
    Q8Cache cache; Q8Seqs seq;
    const __half* q; long long q_stride;
    const int* q_offsets;          // or nullptr: one row each
    int total_q, max_q, max_seq;
    int qpk, window, sinks;        // window 0x7fffffff: none
    float scale_log2;              // scale * log2(e)
    float* mass; int mass_width;
    float2* page_ws; int ws_tiles; // mass: (sum, maximum) of every visited 16-token tile, per row
    float2* part_ml; float* part_o; // parts without a cluster: state and accumulators of every (unit, part)
    float* out; __half* out_h;
    int parts, chunk, cluster;     // parts a unit's tiles are cut into, of `chunk` tiles each; whether they form a cluster
    int row_blocks, row_block0;
};
// The keys a block of query rows sees: [0, sinks) and [low, end), as 16-token tiles.
struct View {
    int len, n;          // tokens, query rows' tokens
    int pos0, pos1;      // positions of the block's first and last query token
    int low0, low1;      // first windowed key of those two
    int end;             // keys [0, end) are at most seen
    int paged;           // tokens held in pages
    int ns, w0, tiles;   // page tiles: 0 .. ns - 1, then w0 ..; `tiles` in all
    int tail_tiles;
};
__device__ __forceinline__ View make_view(const Q8AttnParams& p, int len, int n, int tok0, int tok1) {
    View v;
    v.len = len; v.n = n;
    v.pos0 = len - n + tok0; v.pos1 = len - n + tok1;
    v.low0 = max(0, p.window == 0x7fffffff ? 0 : v.pos0 - p.window + 1);
    v.low1 = max(0, p.window == 0x7fffffff ? 0 : v.pos1 - p.window + 1);
    v.end = max(0, v.pos1 + 1);
    v.paged = len >> p.cache.log2b << p.cache.log2b;
    const int qt = (min(v.end, v.paged) + 15) >> 4;
    v.ns = min((min(p.sinks, v.low0) + 15) >> 4, qt);
    v.w0 = min(v.low0 >> 4, qt);
    if (v.ns >= v.w0) { v.ns = 0; v.w0 = 0; }
    v.tiles = v.ns + qt - v.w0;
    v.tail_tiles = v.end > v.paged ? (v.end - v.paged + 15) >> 4 : 0;
    return v;
}

// One (sequence, kv head, block of R query rows).
struct Unit {
    int seq, h, rb, len, n, row0, rows;
    View v;
    int items;          // tiles of the page part and of the tail
    bool refused;       // its query rows do not lie inside the launch's
    bool counted;       // refused, or its length had to be brought into the launch's bounds
};
__device__ __forceinline__ Unit make_unit(const Q8AttnParams& p, int unit, int r_per_block) {
    Unit u;
    u.rb = unit % p.row_blocks + p.row_block0;
    unit /= p.row_blocks;
    u.h = unit % p.cache.nkv; u.seq = unit / p.cache.nkv;
    const int len = p.seq.lens[u.seq];
    u.len = min(max(len, 0), p.max_seq);
    u.row0 = u.seq; u.n = 1;
    u.refused = false;
    if (p.q_offsets) {
        u.row0 = p.q_offsets[u.seq];
        u.n = p.q_offsets[u.seq + 1] - u.row0;
        if (u.row0 < 0 || u.n < 0 || u.n > p.max_q || u.row0 > p.total_q - u.n) { u.n = 0; u.refused = true; }
    }
    u.counted = u.refused || u.len != len;
    u.rows = u.n * p.qpk;
    const int first = u.rb * r_per_block, last = min(first + r_per_block, u.rows) - 1;
    u.v = make_view(p, u.len, u.n, first / p.qpk, max(last, 0) / p.qpk);
    u.items = u.v.tiles + u.v.tail_tiles;
    return u;
}

// Where row `row` of a unit's output starts, in elements.
__device__ __forceinline__ size_t out_at(const Q8AttnParams& p, const Unit& u, int row, int d) {
    return ((size_t)(u.row0 + row / p.qpk) * p.cache.nkv * p.qpk + u.h * p.qpk + row % p.qpk) * d;
}
constexpr float kQ8Unset = -3.0e38f;     // running maximum before any visible token
constexpr float kQ8Lazy = 8.0f;          // the maximum is raised when a score tops it by 2^8
constexpr float kQ8Headroom = 64.0f;     // probabilities in fp16 carry 2^6: p vs <= 2^8 2^6 < 65504, 2^20 below 1 stay normal

struct Q8EvictParams {
    const int* tables; int width;
    const int* lens; const float* mass; int mass_width;
    int nkv, log2b, batch, max_seq, budget, first, recent;
    int* new_tables; int* new_lens; float* new_mass; int* freed; int* freed_counts;
};
cudaError_t launch_q8_gather(const int* tables, int width, const int* lens, bool by_slot, int rows, const int* slots, int batch,
                             int* out_tables, int* out_lens, cudaStream_t stream);
cudaError_t launch_q8_advance(int* lens, int rows, const int* slots, const int* offsets, int batch, cudaStream_t stream);
cudaError_t launch_q8_write(const Q8WriteParams& p, int d, int fmt, cudaStream_t stream);
cudaError_t launch_q8_read(const Q8ReadParams& p, int d, int fmt, cudaStream_t stream);
cudaError_t launch_q8_attention(const Q8AttnParams& p, int d, int fmt, void* workspace, cudaStream_t stream);
size_t q8_attention_workspace(int nkv, int qpk, int d, int block, int batch, int max_q, int max_seq, int window, int sinks, bool mass);
cudaError_t launch_q8_prompt(const Q8AttnParams& p, int d, int fmt, cudaStream_t stream);
cudaError_t q8_prompt_failures(unsigned int* count);
cudaError_t launch_q8_evict(const Q8EvictParams& p, cudaStream_t stream);
int q8_evict_max_pages();

}  // namespace kivi
