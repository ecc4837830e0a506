// Eviction from a paged cache by accumulated attention weight: which complete pages of a sequence stay, and the
// tables, masses and freed ids that follow.
//
// Per sequence: rank = fp32(sum over kv heads of page_mass, in 64 bits), keep the protected pages and the `budget`
// minus those highest-ranking others (equal: lowest index first). A sequence whose length lies outside the bounds goes
// through as it is: cutting it would lose the pages behind the bound. One CTA per sequence holds the ranks as ordered
// 32-bit keys in shared memory, finds the smallest kept key by a four-pass radix selection, and closes the kept pages
// up with a running prefix count. Bound by latency: a few thousand keys, each read once from HBM and written once.
// Measured: 4 sequences of 2048 tokens 8.8 us, 128 of 9000 .. 32768 tokens 13.8 us (2.6 us of data); with one atomic per
// key and a serial search of the digits 29 and 33 us.
#include "q8_common.cuh"

namespace kivi {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxKeys = 48 * 1024;   // pages of a sequence the shared memory holds a 4-byte key for

__device__ unsigned int g_q8_evict_rejected;

// Larger floats have larger keys; -0 equals 0; NaN is 0, below -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0u;
    x += 0.0f;
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix count of a flag over the CTA and the total; all threads call it.
__device__ __forceinline__ int prefix_of(bool flag, int* warp_sums, int& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned ballot = __ballot_sync(0xffffffffu, flag);
    if (lane == 0) warp_sums[warp] = __popc(ballot);
    __syncthreads();
    const int mine = warp_sums[lane];     // 32 warps
    int before = lane < warp ? mine : 0, all = mine;
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    __syncthreads();
    total = all;
    return before + __popc(ballot & ((1u << lane) - 1u));
}

__global__ void __launch_bounds__(kThreads) q8_evict_kernel(const Q8EvictParams p) {
    extern __shared__ uint32_t keys[];    // then, in its place, the kept pages in order
    __shared__ int hist[256];
    __shared__ int warp_sums[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int seq = blockIdx.x, tid = threadIdx.x;
    const int* table = p.tables + (size_t)seq * p.width;
    int* new_table = p.new_tables + (size_t)seq * p.width;
    int* freed = p.freed + (size_t)seq * p.width;
    const float* mass = p.mass + (size_t)seq * p.nkv * p.mass_width;
    float* new_mass = p.new_mass + (size_t)seq * p.nkv * p.mass_width;
    const int len = p.lens[seq];
    if (len < 0 || len > p.max_seq) {     // (max_seq's pages fit the table and the masses)
        for (int i = tid; i < p.width; i += kThreads) { new_table[i] = table[i]; freed[i] = -1; }
        for (size_t i = tid; i < (size_t)p.nkv * p.mass_width; i += kThreads) new_mass[i] = mass[i];
        if (tid == 0) { p.new_lens[seq] = len; p.freed_counts[seq] = 0; atomicAdd(&g_q8_evict_rejected, 1u); }
        return;
    }
    const int full = len >> p.log2b, open = len & ((1 << p.log2b) - 1);
    const bool all = full <= p.budget;
    const int lo = min(p.first, full), hi = max(lo, full - p.recent);   // candidates [lo, hi)
    uint32_t threshold = 0;
    int ties = 0;                          // candidates with exactly the threshold's key that stay
    if (!all) {
        for (int i = lo + tid; i < hi; i += kThreads) {
            double sum = 0.0;
            for (int h0 = 0; h0 < p.nkv; h0 += 8) {   // eight heads' loads in flight, added in order
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = h0 + k < p.nkv ? mass[(size_t)(h0 + k) * p.mass_width + i] : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += (double)x[k];
            }
            keys[i] = key_of((float)sum);
        }
        // budget < full and first + recent <= budget, so 0 <= need < hi - lo
        if (tid == 0) { s_prefix = 0; s_need = p.budget - lo - (full - hi); }
        __syncthreads();
        const int need = p.budget - lo - (full - hi);
        // the need-th largest key, byte by byte (need = 0: nothing but the protected pages stays)
        for (int shift = 24; need > 0 && shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
            // masses share their leading bits: one atomic per distinct digit of a warp, not per key
            for (int base = lo; base < hi; base += kThreads) {
                const int i = base + tid;
                const bool in = i < hi && (keys[i] & mask) == prefix;
                const int digit = in ? (int)(keys[i] >> shift) & 255 : 256;
                const unsigned same = __match_any_sync(0xffffffffu, digit);
                if (in && (tid & 31) == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
            }
            __syncthreads();
            if (tid < 32) {   // from the highest digit down: lane l counts digits 255 - 8 l .. 248 - 8 l
                int mine = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) mine += hist[255 - 8 * tid - k];
                int upto = mine;
#pragma unroll
                for (int x = 1; x < 32; x *= 2) {
                    const int y = __shfl_up_sync(0xffffffffu, upto, x);
                    if (tid >= x) upto += y;
                }
                const int want = s_need;
                __syncwarp();
                if (want > upto - mine && want <= upto) {   // exactly one lane, as 1 <= want <= all
                    int left = want - (upto - mine), b = 255 - 8 * tid;
                    while (hist[b] < left) left -= hist[b--];
                    s_need = left;
                    s_prefix = prefix | ((uint32_t)b << shift);
                }
            }
            __syncthreads();
        }
        threshold = s_prefix;
        ties = s_need;
        if (need == 0) { threshold = 0xffffffffu; ties = 0; }
    }
    // close up, in order
    int kept = 0, gone = 0, tied = 0;
    for (int base = 0; base < full; base += kThreads) {
        const int i = base + tid;
        const bool here = i < full, fixed = here && (all || i < lo || i >= hi);
        const uint32_t key = here && !fixed ? keys[i] : 0u;
        int total;
        const bool tie = here && !fixed && key == threshold;
        const int before = tied + prefix_of(tie, warp_sums, total);
        tied += total;
        const bool keep = fixed || (here && !fixed && (key > threshold || (tie && before < ties)));
        const int at = kept + prefix_of(keep, warp_sums, total);
        kept += total;
        const bool out = here && !keep;
        const int at_gone = gone + prefix_of(out, warp_sums, total);
        gone += total;
        // prefix_of has barriers behind every read of keys[base ..], and at <= i: nothing unread is overwritten
        if (keep) { keys[at] = (uint32_t)i; new_table[at] = table[i]; }
        if (out) freed[at_gone] = table[i];
    }
    __syncthreads();
    for (int i = kept + tid; i < p.width; i += kThreads) new_table[i] = 0;
    for (int i = gone + tid; i < p.width; i += kThreads) freed[i] = -1;
    if (tid == 0) {
        p.new_lens[seq] = (kept << p.log2b) + open;
        p.freed_counts[seq] = gone;
    }
    const int columns = kept + (open && full < p.mass_width ? 1 : 0);   // the open block's mass moves up behind them
    for (int h = 0; h < p.nkv; ++h)
        for (int i = tid; i < p.mass_width; i += kThreads)
            new_mass[(size_t)h * p.mass_width + i] =
                i < columns ? mass[(size_t)h * p.mass_width + (i < kept ? (int)keys[i] : full)] : 0.0f;
}

}  // namespace

cudaError_t q8_evict_rejected(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_q8_evict_rejected, sizeof(*count)); }

int q8_evict_max_pages() { return kMaxKeys; }

cudaError_t launch_q8_evict(const Q8EvictParams& p, cudaStream_t stream) {
    const size_t smem = sizeof(uint32_t) * (size_t)(p.width < 1 ? 1 : p.width);
    static Q8SmemLimit limit;
    const cudaError_t e = limit.raise(q8_evict_kernel, (int)(kMaxKeys * sizeof(uint32_t)));
    if (e != cudaSuccess) return e;
    q8_evict_kernel<<<p.batch, kThreads, smem, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace kivi
