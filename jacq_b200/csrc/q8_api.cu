// C entry points of the 8-bit block-scaled cache: argument checks before anything is launched.
#include "q8_common.cuh"

namespace kivi {
namespace {

bool q8_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int q8_log2(int block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : -1; }

int check_q8_geometry(const kivi_q8_geometry* g) {
    if (!g) return KIVI_ERR_NULL_POINTER;
    if (g->num_q_heads <= 0 || g->num_kv_heads <= 0 || g->num_q_heads % g->num_kv_heads || g->num_q_heads > 32767) return KIVI_ERR_GEOMETRY;
    if (g->head_dim != 64 && g->head_dim != 128 && g->head_dim != 256) return KIVI_ERR_GEOMETRY;
    if (q8_log2(g->block_size) < 0) return KIVI_ERR_GEOMETRY;
    if (g->format != KIVI_Q8_INT8 && g->format != KIVI_Q8_E4M3) return KIVI_ERR_GEOMETRY;
    return KIVI_OK;
}

int check_q8_cache(const kivi_q8_cache* c) {
    if (!c) return KIVI_ERR_NULL_POINTER;
    const void* ptrs[] = {c->k_pages, c->v_pages, c->scales, c->k_tail, c->v_tail};
    for (const void* p : ptrs) {
        if (!p) return KIVI_ERR_NULL_POINTER;
        if (!q8_aligned16(p)) return KIVI_ERR_ALIGNMENT;
    }
    if (c->num_blocks <= 0 || c->num_slots <= 0) return KIVI_ERR_RANGE;
    return KIVI_OK;
}

Q8Cache q8_cache_of(const kivi_q8_geometry& g, const kivi_q8_cache& c) {
    Q8Cache o;
    o.k = c.k_pages; o.v = c.v_pages;
    o.scales = reinterpret_cast<float2*>(c.scales);
    o.k_tail = reinterpret_cast<__half*>(c.k_tail); o.v_tail = reinterpret_cast<__half*>(c.v_tail);
    o.num_blocks = c.num_blocks; o.num_slots = c.num_slots;
    o.nkv = g.num_kv_heads; o.log2b = q8_log2(g.block_size);
    return o;
}

constexpr int kQ8MaxLen = (1 << 30) - 1;
constexpr int kQ8MaxBatch = 65535;   // one grid dimension of the writer

// What all calls check of a batch: the tables and the slots.
int check_q8_batch(const kivi_q8_cache* cache, const int32_t* tables, int width, const int32_t* slot_ids, int batch) {
    if (batch < 0 || batch > kQ8MaxBatch || width < 0) return KIVI_ERR_RANGE;
    if (!tables && width > 0 && batch > 0) return KIVI_ERR_NULL_POINTER;
    if (!slot_ids && batch > cache->num_slots) return KIVI_ERR_RANGE;
    return KIVI_OK;
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" int kivi_b200_q8_validate_geometry(const kivi_q8_geometry* geom) { return check_q8_geometry(geom); }

extern "C" int kivi_b200_q8_gather_slots(const int32_t* block_tables, int max_blocks_per_seq, const int32_t* seq_lens, int lens_by_slot,
                                         int num_rows, const int32_t* slot_ids, int batch, int32_t* out_tables, int32_t* out_lens,
                                         cudaStream_t stream) {
    if (batch < 0 || batch > kQ8MaxBatch || max_blocks_per_seq < 0 || num_rows < 0) return KIVI_ERR_RANGE;
    if (batch == 0) return KIVI_OK;
    if (!slot_ids || !out_lens || (!seq_lens && num_rows) || (max_blocks_per_seq && (!out_tables || (!block_tables && num_rows))))
        return KIVI_ERR_NULL_POINTER;
    return launch_q8_gather(block_tables, max_blocks_per_seq, seq_lens, lens_by_slot != 0, num_rows, slot_ids, batch, out_tables,
                            out_lens, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

extern "C" int kivi_b200_q8_advance_slots(int32_t* seq_lens, int num_rows, const int32_t* slot_ids, const int32_t* new_offsets,
                                          int batch, cudaStream_t stream) {
    if (batch < 0 || batch > kQ8MaxBatch || num_rows < 0) return KIVI_ERR_RANGE;
    if (batch == 0 || num_rows == 0) return KIVI_OK;
    if (!seq_lens || !slot_ids || !new_offsets) return KIVI_ERR_NULL_POINTER;
    return launch_q8_advance(seq_lens, num_rows, slot_ids, new_offsets, batch, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

extern "C" int kivi_b200_q8_cache_write(const kivi_q8_geometry* geom, const kivi_q8_cache* cache, const kivi_f16* new_k,
                                        const kivi_f16* new_v, int64_t k_stride, int64_t v_stride,
                                        const int32_t* block_tables, int max_blocks_per_seq, const int32_t* start_seq_lens,
                                        const int32_t* new_offsets, const int32_t* slot_ids, int batch, int total_new,
                                        int max_new_per_seq, int max_start_seq_len, cudaStream_t stream) {
    int rc = check_q8_geometry(geom);
    if (rc == KIVI_OK) rc = check_q8_cache(cache);
    if (rc == KIVI_OK) rc = check_q8_batch(cache, block_tables, max_blocks_per_seq, slot_ids, batch);
    if (rc != KIVI_OK) return rc;
    if (total_new < 0 || max_new_per_seq < 0 || max_start_seq_len < 0 || max_new_per_seq > kQ8MaxLen - 128 ||
        max_start_seq_len > kQ8MaxLen) return KIVI_ERR_RANGE;
    if (batch == 0 || total_new == 0 || max_new_per_seq == 0) return KIVI_OK;
    if (!new_k || !new_v || !start_seq_lens || !new_offsets) return KIVI_ERR_NULL_POINTER;
    if (!q8_aligned16(new_k) || !q8_aligned16(new_v) || k_stride % 8 || v_stride % 8) return KIVI_ERR_ALIGNMENT;
    const int64_t row = (int64_t)geom->num_kv_heads * geom->head_dim;
    if (k_stride < row || v_stride < row) return KIVI_ERR_RANGE;
    Q8WriteParams p;
    p.cache = q8_cache_of(*geom, *cache);
    p.seq = Q8Seqs{block_tables, max_blocks_per_seq, start_seq_lens, slot_ids, batch};
    p.new_k = reinterpret_cast<const __half*>(new_k); p.new_v = reinterpret_cast<const __half*>(new_v);
    p.k_stride = k_stride; p.v_stride = v_stride;
    p.offsets = new_offsets; p.total_new = total_new; p.max_new = max_new_per_seq; p.max_start = max_start_seq_len;
    return launch_q8_write(p, geom->head_dim, geom->format, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

extern "C" int kivi_b200_q8_cache_read(const kivi_q8_geometry* geom, const kivi_q8_cache* cache, const int32_t* block_tables,
                                       int max_blocks_per_seq, const int32_t* seq_lens, const int32_t* slot_ids,
                                       const int32_t* row_offsets, const int32_t* first_rows, int batch, int total_rows,
                                       int max_rows_per_seq, kivi_f16* k_out, kivi_f16* v_out, cudaStream_t stream) {
    int rc = check_q8_geometry(geom);
    if (rc == KIVI_OK) rc = check_q8_cache(cache);
    if (rc == KIVI_OK) rc = check_q8_batch(cache, block_tables, max_blocks_per_seq, slot_ids, batch);
    if (rc != KIVI_OK) return rc;
    if (total_rows < 0 || max_rows_per_seq < 0 || max_rows_per_seq > kQ8MaxLen) return KIVI_ERR_RANGE;
    if (batch == 0 || total_rows == 0 || max_rows_per_seq == 0) return KIVI_OK;
    if (!seq_lens || !row_offsets || !first_rows || !k_out || !v_out) return KIVI_ERR_NULL_POINTER;
    if (!q8_aligned16(k_out) || !q8_aligned16(v_out)) return KIVI_ERR_ALIGNMENT;
    Q8ReadParams p;
    p.cache = q8_cache_of(*geom, *cache);
    p.seq = Q8Seqs{block_tables, max_blocks_per_seq, seq_lens, slot_ids, batch};
    p.offsets = row_offsets; p.first = first_rows;
    p.total_rows = total_rows; p.max_rows = max_rows_per_seq;
    p.k_out = reinterpret_cast<__half*>(k_out); p.v_out = reinterpret_cast<__half*>(v_out);
    return launch_q8_read(p, geom->head_dim, geom->format, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

namespace {
constexpr int kNoWindow = 0x7fffffff;
// A window of max_seq_len tokens or more hides none; as a number it would overflow in positions before the first token.
int window_of(int window, int max_seq) { return window == 0 || window >= max_seq ? kNoWindow : window; }
// Grid size of a call: (sequence, kv head, block of 8 query rows) units cut into at most 32 parts.
bool q8_grid_fits(const kivi_q8_geometry* g, int batch, int max_q) {
    const int64_t rows = (int64_t)max_q * (g->num_q_heads / g->num_kv_heads);
    return rows < (1 << 24) && (int64_t)batch * g->num_kv_heads * ((rows + 7) / 8) < (1LL << 27);
}
}  // namespace

extern "C" size_t kivi_b200_q8_attention_workspace_bytes(const kivi_q8_geometry* geom, int batch, int max_q_per_seq,
                                                         int max_seq_len, int window, int sinks, int with_mass) {
    if (check_q8_geometry(geom) != KIVI_OK || batch < 1 || batch > kQ8MaxBatch || max_q_per_seq < 1 || max_seq_len < 0 ||
        max_seq_len > kQ8MaxLen || window < 0 || sinks < 0 || !q8_grid_fits(geom, batch, max_q_per_seq)) return 0;
    return q8_attention_workspace(geom->num_kv_heads, geom->num_q_heads / geom->num_kv_heads, geom->head_dim, geom->block_size, batch, max_q_per_seq,
                                  max_seq_len, window_of(window, max_seq_len), sinks, with_mass != 0);
}

extern "C" int kivi_b200_q8_attention(const kivi_q8_geometry* geom, const kivi_q8_cache* cache, const kivi_f16* q,
                                      int64_t q_stride, const int32_t* q_offsets, int total_q, const int32_t* block_tables,
                                      int max_blocks_per_seq, const int32_t* seq_lens, const int32_t* slot_ids, int batch,
                                      int max_q_per_seq, int max_seq_len, int window, int sinks, float scale,
                                      float* page_mass, int mass_width, float* out_f32, kivi_f16* out_f16, void* workspace,
                                      size_t workspace_bytes, cudaStream_t stream) {
    int rc = check_q8_geometry(geom);
    if (rc == KIVI_OK) rc = check_q8_cache(cache);
    if (rc == KIVI_OK) rc = check_q8_batch(cache, block_tables, max_blocks_per_seq, slot_ids, batch);
    if (rc != KIVI_OK) return rc;
    if (total_q < 0 || max_q_per_seq < 0 || max_seq_len < 0 || max_seq_len > kQ8MaxLen || window < 0 || sinks < 0 ||
        !(scale >= 0.0f && scale < 1e30f)) return KIVI_ERR_RANGE;
    if (batch == 0 || total_q == 0 || max_q_per_seq == 0) return KIVI_OK;
    if (!q || !seq_lens || (!out_f32 && !out_f16)) return KIVI_ERR_NULL_POINTER;
    if (out_f32 && out_f16) return KIVI_ERR_RANGE;
    if (!q_offsets && (total_q != batch || max_q_per_seq != 1)) return KIVI_ERR_RANGE;
    if (!q8_aligned16(q) || q_stride % 8 || !q8_aligned16(out_f32) || !q8_aligned16(out_f16)) return KIVI_ERR_ALIGNMENT;
    if (q_stride < (int64_t)geom->num_q_heads * geom->head_dim || !q8_grid_fits(geom, batch, max_q_per_seq)) return KIVI_ERR_RANGE;
    if (max_seq_len / geom->block_size > max_blocks_per_seq) return KIVI_ERR_BLOCK_TABLE;
    Q8AttnParams p = {};
    p.cache = q8_cache_of(*geom, *cache);
    p.seq = Q8Seqs{block_tables, max_blocks_per_seq, seq_lens, slot_ids, batch};
    p.q = reinterpret_cast<const __half*>(q); p.q_stride = q_stride; p.q_offsets = q_offsets;
    p.total_q = total_q; p.max_q = max_q_per_seq; p.max_seq = max_seq_len;
    p.qpk = geom->num_q_heads / geom->num_kv_heads;
    p.window = window_of(window, max_seq_len); p.sinks = sinks;
    const float s = scale > 0.0f ? scale : (geom->head_dim == 64 ? 0.125f : geom->head_dim == 256 ? 0.0625f : 0.08838834764831845f);
    p.scale_log2 = s * 1.4426950408889634f;
    p.out = out_f32; p.out_h = reinterpret_cast<__half*>(out_f16);
    if (page_mass) {
        if (q_offsets) return KIVI_ERR_RANGE;
        if ((int64_t)mass_width * geom->block_size < max_seq_len) return KIVI_ERR_RANGE;
        p.mass = page_mass; p.mass_width = mass_width;
    }
    const size_t need = q8_attention_workspace(geom->num_kv_heads, p.qpk, geom->head_dim, geom->block_size, batch, max_q_per_seq, max_seq_len, p.window,
                                               sinks, page_mass != nullptr);
    if (need) {
        if (!workspace || workspace_bytes < need) return KIVI_ERR_WORKSPACE;
        if (!q8_aligned16(workspace)) return KIVI_ERR_ALIGNMENT;
    }
    return launch_q8_attention(p, geom->head_dim, geom->format, workspace, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

extern "C" int kivi_b200_q8_evict(int num_kv_heads, int block_size, const int32_t* block_tables, int max_blocks_per_seq,
                                  const int32_t* seq_lens, const float* page_mass, int mass_width, int batch, int max_seq_len,
                                  int budget, int first, int recent, int32_t* new_tables, int32_t* new_lens, float* new_mass,
                                  int32_t* freed, int32_t* freed_counts, cudaStream_t stream) {
    if (num_kv_heads < 1 || q8_log2(block_size) < 0) return KIVI_ERR_GEOMETRY;
    if (batch < 0 || batch > kQ8MaxBatch || max_blocks_per_seq < 1 || max_blocks_per_seq > q8_evict_max_pages() || mass_width < 0 ||
        max_seq_len < 0 || max_seq_len > kQ8MaxLen || budget < 0 || first < 0 || recent < 0 || (int64_t)first + recent > budget)
        return KIVI_ERR_RANGE;
    if ((int64_t)mass_width * block_size < max_seq_len) return KIVI_ERR_RANGE;
    if (max_seq_len / block_size > max_blocks_per_seq) return KIVI_ERR_BLOCK_TABLE;
    if (batch == 0) return KIVI_OK;
    if (!block_tables || !seq_lens || (!page_mass && mass_width) || !new_tables || !new_lens || (!new_mass && mass_width) || !freed ||
        !freed_counts) return KIVI_ERR_NULL_POINTER;
    if (new_tables == block_tables || new_lens == seq_lens || (new_mass == page_mass && mass_width) || freed == block_tables || freed == new_tables)
        return KIVI_ERR_RANGE;
    Q8EvictParams p;
    p.tables = block_tables; p.width = max_blocks_per_seq;
    p.lens = seq_lens; p.mass = page_mass; p.mass_width = mass_width;
    p.nkv = num_kv_heads; p.log2b = q8_log2(block_size); p.batch = batch; p.max_seq = max_seq_len;
    p.budget = budget; p.first = first; p.recent = recent;
    p.new_tables = new_tables; p.new_lens = new_lens; p.new_mass = new_mass; p.freed = freed; p.freed_counts = freed_counts;
    return launch_q8_evict(p, stream) == cudaSuccess ? KIVI_OK : KIVI_ERR_CUDA;
}

extern "C" int kivi_b200_q8_rejected_indices(uint32_t* count_out) {
    if (!count_out) return KIVI_ERR_NULL_POINTER;
    unsigned int a = 0, b = 0, c = 0, d = 0;
    if (q8_cache_rejected(&a) != cudaSuccess || q8_attention_rejected(&b) != cudaSuccess || q8_prompt_rejected(&c) != cudaSuccess ||
        q8_evict_rejected(&d) != cudaSuccess)
        return KIVI_ERR_CUDA;
    *count_out = a + b + c + d;
    return KIVI_OK;
}

extern "C" int kivi_b200_q8_wait_failures(uint32_t* count_out) {
    if (!count_out) return KIVI_ERR_NULL_POINTER;
    unsigned int n = 0;
    if (q8_prompt_failures(&n) != cudaSuccess) return KIVI_ERR_CUDA;
    *count_out = n;
    return KIVI_OK;
}
