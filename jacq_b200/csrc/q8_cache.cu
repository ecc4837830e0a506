// Writer and read-back of the 8-bit block-scaled cache.
//
// Writer: scale = max|x| * fp32(1 / top), code = rne(x / scale) over the B x D values of a block, top = 127 (int8) or
// 448 (e4m3). Bound by HBM: 2 bytes in and 1 byte out per value. A warp holds 16 token rows of one head in registers
// (16 x D fp16, 32 registers per lane at D = 128), so the block is read once: the extreme is found in registers, across
// the B / 16 warps of a block through shared memory, and the codes are made from the same registers. Measured: 96
// prompts of 1 .. 1024 tokens, 8 heads of 128, e4m3, written and read back: 110 us, 5.2 TB/s, 0.81 of the copy rate.
#include "q8_common.cuh"

namespace kivi {
namespace {

__device__ unsigned int g_q8_cache_rejected;

// fp32 quotient a / s from y = RN(1 / s): q0 = a y, then one correction by its exact remainder, which gives the
// correctly rounded quotient (Markstein's theorem; no under- or overflow: a and s come from fp16 values).
__device__ __forceinline__ float quotient(float a, float s, float y) {
    const float q0 = a * y;
    return __fmaf_rn(__fmaf_rn(-s, q0, a), y, q0);
}

template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FMT == KIVI_Q8_INT8) {
        // 1.5 * 2^23 added: the low byte of the sum's bits is the rounded value in two's complement
        const uint32_t x = __float_as_uint(a + 12582912.0f), y = __float_as_uint(b + 12582912.0f);
        const uint32_t z = __float_as_uint(c + 12582912.0f), w = __float_as_uint(d + 12582912.0f);
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    } else {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
}

// What a sequence of the launch writes: `start` tokens before, `n` new rows from `row0` on.
struct WriteSpan { int start, n, row0, slot; bool ok; };

__device__ __forceinline__ WriteSpan write_span(const Q8WriteParams& p, int i) {
    WriteSpan w;
    w.start = p.seq.lens[i];
    w.row0 = p.offsets[i];
    w.n = p.offsets[i + 1] - w.row0;
    w.slot = q8_slot(p.seq, i);
    const long long end = (long long)w.start + w.n;
    w.ok = w.start >= 0 && w.start <= p.max_start && w.n >= 0 && w.n <= p.max_new && w.row0 >= 0 &&
           w.row0 <= p.total_new - w.n && index_in_pool(w.slot, p.cache.num_slots) && end < (1LL << 30) &&
           (end >> p.cache.log2b) <= p.seq.width;
    return w;
}

// Whether all pages a sequence would complete lie in the pool (its threads share the ids; uniform over the CTA).
__device__ __forceinline__ bool pages_ok(const Q8WriteParams& p, int i, const WriteSpan& w) {
    bool ok = w.ok;
    if (ok) {
        const int b0 = w.start >> p.cache.log2b, b1 = (w.start + w.n) >> p.cache.log2b;
        const int* row = p.seq.tables + (size_t)i * p.seq.width;
        for (int b = b0 + threadIdx.x; b < b1; b += blockDim.x) ok &= index_in_pool(row[b], p.cache.num_blocks);
    }
    return __syncthreads_and(ok);
}

// One CTA: kWarps / WPB blocks of one (sequence, head, K | V); WPB = B / 16 warps hold a block. The unit that holds the
// sequence's first touched block also moves what stays in fp16 to the tail rows: it is the only one that reads old
// tail rows, and it has them in registers before it writes new ones.
template <int D, int FMT>
__global__ void __launch_bounds__(256) q8_write_kernel(const Q8WriteParams p, int wpb) {
    constexpr int LPR = D / 8;             // lanes per row, 8 values (16 bytes) each
    constexpr int RPI = 32 / LPR;          // rows a warp instruction covers
    constexpr int NI = 16 / RPI;           // instructions for 16 rows
    __shared__ float warp_max[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int nkv = p.cache.nkv, block = 1 << p.cache.log2b;
    const int hw = blockIdx.y, h = hw >> 1, which = hw & 1;
    const int i = blockIdx.z;
    const WriteSpan w = write_span(p, i);
    if (!pages_ok(p, i, w)) {
        if (blockIdx.x == 0 && hw == 0 && threadIdx.x == 0) atomicAdd(&g_q8_cache_rejected, 1u);
        return;
    }
    if (w.n == 0) return;
    const int b0 = w.start >> p.cache.log2b, had = w.start & (block - 1);
    const int full = (had + w.n) >> p.cache.log2b;          // blocks that become complete
    const int ord = blockIdx.x * (warps / wpb) + warp / wpb;  // which of them this warp's block is
    if (blockIdx.x * (warps / wpb) > (full ? full - 1 : 0)) return;   // uniform over the CTA
    const __half* src = which ? p.new_v : p.new_k;
    const long long stride = which ? p.v_stride : p.k_stride;
    __half* tail = (which ? p.cache.v_tail : p.cache.k_tail) + ((size_t)w.slot * nkv + h) * block * D;
    const int r0 = (warp % wpb) * 16 + lane / LPR, c0 = (lane % LPR) * 8;
    const __half* src_c = src + (size_t)h * D + c0;
    const bool mine = ord < full;
    uint4 x[NI];
    if (mine) {
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            const int row = r0 + k * RPI, tok = ord * block + row;  // tok: counted from the open block's first token
            x[k] = tok < had ? *reinterpret_cast<const uint4*>(tail + (size_t)row * D + c0)
                             : __ldcs(reinterpret_cast<const uint4*>(src_c + (long long)(w.row0 + tok - had) * stride));
        }
        __half2 top = __float2half2_rn(0.0f);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            const __half2* e = reinterpret_cast<const __half2*>(&x[k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) top = __hmax2_nan(top, __habs2(e[j]));
        }
        // NaN stays NaN through the maxima; as unsigned bits it is above every number
        uint32_t t = max(__half_as_ushort(__low2half(top)), __half_as_ushort(__high2half(top)));
        t = __reduce_max_sync(0xffffffffu, t);
        if (lane == 0) warp_max[warp] = __half2float(__ushort_as_half((unsigned short)t));
        if (lane == 0 && t >= 0x7c00u) warp_max[warp] = __int_as_float(0x7f800000);   // any infinity or NaN: one mark
    }
    __syncthreads();
    if (mine) {
        float top = 0.0f;
        for (int k = 0; k < wpb; ++k) top = fmaxf(top, warp_max[warp / wpb * wpb + k]);
        const bool finite = top < 1e30f;
        const float scale = finite ? top * (FMT == KIVI_Q8_INT8 ? kQ8RecipInt8 : kQ8RecipE4m3) : __int_as_float(0x7fc00000);
        const bool live = finite && top > 0.0f;
        const float rcp = live ? __frcp_rn(scale) : 0.0f;
        const int id = p.seq.tables[(size_t)i * p.seq.width + b0 + ord];
        const size_t page = (size_t)id * nkv + h;
        uint8_t* dst = (which ? p.cache.v : p.cache.k) + page * block * D;
        if (warp % wpb == 0 && lane == 0) reinterpret_cast<float*>(p.cache.scales + page)[which] = scale;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            uint2 code = make_uint2(0u, 0u);
            if (live) {
                const __half2* e = reinterpret_cast<const __half2*>(&x[k]);
                float q[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(e[j]);
                    q[2 * j] = quotient(f.x, scale, rcp);
                    q[2 * j + 1] = quotient(f.y, scale, rcp);
                    if constexpr (FMT == KIVI_Q8_E4M3) {   // the correction turns -0 into 0, and e4m3 has both
                        q[2 * j] = copysignf(q[2 * j], f.x);
                        q[2 * j + 1] = copysignf(q[2 * j + 1], f.y);
                    }
                }
                code.x = encode4<FMT>(q[0], q[1], q[2], q[3]);
                code.y = encode4<FMT>(q[4], q[5], q[6], q[7]);
            }
            *reinterpret_cast<uint2*>(dst + (size_t)(r0 + k * RPI) * D + c0) = code;
        }
    }
    // the rows that stay: new rows behind the last complete block
    if (blockIdx.x != 0) return;
    const int keep = (had + w.n) & (block - 1), from = full ? 0 : had;
    for (int row = from + warp * RPI + lane / LPR; row < keep; row += warps * RPI) {
        const int tok = full * block + row;
        *reinterpret_cast<uint4*>(tail + (size_t)row * D + c0) =
            *reinterpret_cast<const uint4*>(src_c + (long long)(w.row0 + tok - had) * stride);
    }
}

// Read-back: 16 rows of one head per warp, values code * scale rounded to fp16 (tail rows as they are). Bound by HBM:
// 1 byte in, 2 bytes out per value.
template <int D, int FMT>
__global__ void __launch_bounds__(256) q8_read_kernel(const Q8ReadParams p) {
    constexpr int LPR = D / 8, RPI = 32 / LPR, NI = 16 / RPI;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nkv = p.cache.nkv, block = 1 << p.cache.log2b;
    const int hw = blockIdx.y, h = hw >> 1, which = hw & 1;
    const int i = blockIdx.z;
    const int len = p.seq.lens[i], row0 = p.offsets[i], first = p.first[i];
    const int n = p.offsets[i + 1] - row0, slot = q8_slot(p.seq, i);
    bool ok = len >= 0 && len < (1 << 30) && first >= 0 && n >= 0 && n <= p.max_rows && row0 >= 0 && row0 <= p.total_rows - n &&
              index_in_pool(slot, p.cache.num_slots) && (len >> p.cache.log2b) <= p.seq.width;
    if (!ok) {
        if (blockIdx.x == 0 && hw == 0 && threadIdx.x == 0) atomicAdd(&g_q8_cache_rejected, 1u);
        return;
    }
    // tiles of 16 tokens, aligned as the pages are
    const int paged = len >> p.cache.log2b << p.cache.log2b;
    const long long end = (long long)first + n;
    const long long t0 = ((long long)(first >> 4) + (long long)blockIdx.x * 8 + warp) << 4;
    if (t0 >= end) return;
    const int r = lane / LPR, c0 = (lane % LPR) * 8;
    const uint8_t* codes = nullptr;
    const __half* rows = nullptr;
    float scale = 0.0f;
    if (t0 >= len) {
        // behind the last token: zeros
    } else if (t0 < paged) {
        const int id = p.seq.tables[(size_t)i * p.seq.width + (t0 >> p.cache.log2b)];
        if (!index_in_pool(id, p.cache.num_blocks)) {
            if (hw == 0 && lane == 0) atomicAdd(&g_q8_cache_rejected, 1u);
            return;
        }
        const size_t page = (size_t)id * nkv + h;
        codes = (which ? p.cache.v : p.cache.k) + (page * block + (t0 & (block - 1))) * D + c0;
        scale = reinterpret_cast<const float*>(p.cache.scales + page)[which];
    } else {
        rows = (which ? p.cache.v_tail : p.cache.k_tail) + (((size_t)slot * nkv + h) * block + (t0 - paged)) * D + c0;
    }
    __half* out = (which ? p.v_out : p.k_out) + (size_t)h * D + c0;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        const int row = r + k * RPI;
        const long long tok = t0 + row;
        if (tok < first || tok >= end) continue;
        uint4 v;
        if (codes) {
            const uint2 w = __ldcs(reinterpret_cast<const uint2*>(codes + (size_t)row * D));
            uint32_t u[4];
            q8_unpack<FMT>(w.x, u[0], u[1]);
            q8_unpack<FMT>(w.y, u[2], u[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
                u[j] = pack_half2(f.x * scale, f.y * scale);
            }
            v = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
            v = tok < len ? *reinterpret_cast<const uint4*>(rows + (size_t)row * D) : make_uint4(0u, 0u, 0u, 0u);
        }
        __stcs(reinterpret_cast<uint4*>(out + ((size_t)row0 + (size_t)(tok - first)) * nkv * D), v);
    }
}

// Rows of per-slot tables and lengths for a batch: one CTA a sequence, bound by its launch.
__global__ void __launch_bounds__(128) q8_gather_kernel(const int* tables, int width, const int* lens, bool by_slot, int rows,
                                                        const int* slots, int* out_tables, int* out_lens) {
    const int i = blockIdx.x, slot = slots[i];
    const bool ok = index_in_pool(slot, rows);
    for (int c = threadIdx.x; c < width; c += 128) out_tables[(size_t)i * width + c] = ok ? tables[(size_t)slot * width + c] : -1;
    if (threadIdx.x == 0) out_lens[i] = ok ? lens[by_slot ? slot : i] : -1;
}
__global__ void __launch_bounds__(128) q8_advance_kernel(int* lens, int rows, const int* slots, const int* offsets, int batch) {
    const int i = blockIdx.x * 128 + threadIdx.x;
    if (i < batch && index_in_pool(slots[i], rows)) atomicAdd(lens + slots[i], offsets[i + 1] - offsets[i]);
}

template <int D>
cudaError_t write_d(const Q8WriteParams& p, int fmt, dim3 grid, int threads, int wpb, cudaStream_t stream) {
    if (fmt == KIVI_Q8_INT8) q8_write_kernel<D, KIVI_Q8_INT8><<<grid, threads, 0, stream>>>(p, wpb);
    else q8_write_kernel<D, KIVI_Q8_E4M3><<<grid, threads, 0, stream>>>(p, wpb);
    return cudaGetLastError();
}
template <int D>
cudaError_t read_d(const Q8ReadParams& p, int fmt, dim3 grid, cudaStream_t stream) {
    if (fmt == KIVI_Q8_INT8) q8_read_kernel<D, KIVI_Q8_INT8><<<grid, 256, 0, stream>>>(p);
    else q8_read_kernel<D, KIVI_Q8_E4M3><<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_q8_gather(const int* tables, int width, const int* lens, bool by_slot, int rows, const int* slots, int batch,
                             int* out_tables, int* out_lens, cudaStream_t stream) {
    q8_gather_kernel<<<batch, 128, 0, stream>>>(tables, width, lens, by_slot, rows, slots, out_tables, out_lens);
    return cudaGetLastError();
}

cudaError_t launch_q8_advance(int* lens, int rows, const int* slots, const int* offsets, int batch, cudaStream_t stream) {
    q8_advance_kernel<<<(batch + 127) / 128, 128, 0, stream>>>(lens, rows, slots, offsets, batch);
    return cudaGetLastError();
}

cudaError_t launch_q8_write(const Q8WriteParams& p, int d, int fmt, cudaStream_t stream) {
    const int block = 1 << p.cache.log2b, wpb = block / 16, warps = wpb > 4 ? wpb : 4;
    const int most = (block - 1 + p.max_new) >> p.cache.log2b;   // blocks a sequence can complete
    const int per = warps / wpb;
    const dim3 grid(most > per ? (most + per - 1) / per : 1, 2 * p.cache.nkv, p.seq.batch);
    switch (d) {
        case 64: return write_d<64>(p, fmt, grid, warps * 32, wpb, stream);
        case 128: return write_d<128>(p, fmt, grid, warps * 32, wpb, stream);
        default: return write_d<256>(p, fmt, grid, warps * 32, wpb, stream);
    }
}

cudaError_t launch_q8_read(const Q8ReadParams& p, int d, int fmt, cudaStream_t stream) {
    const int tiles = (p.max_rows + 15 + 15) / 16;   // an unaligned span touches one tile more
    const dim3 grid((tiles + 7) / 8, 2 * p.cache.nkv, p.seq.batch);
    switch (d) {
        case 64: return read_d<64>(p, fmt, grid, stream);
        case 128: return read_d<128>(p, fmt, grid, stream);
        default: return read_d<256>(p, fmt, grid, stream);
    }
}

cudaError_t q8_cache_rejected(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_q8_cache_rejected, sizeof(*count)); }

}  // namespace kivi
