// Entry points of the attention over a paged cache (paged_attn.cuh), and its bf16 kernels.  The fp16 kernels are a translation unit of their own:
// compiled beside them, which differ in the softmax, the bf16 kernels of 64 dims came out 5 % slower (16 sequences, capped: 16.1 and 17.1 us).
#include "paged_attn.cuh"

namespace nexrt {
template int paged_dispatch<__nv_bfloat16>(const PagedAttnArgs&, int, bool, cudaStream_t);
extern template int paged_dispatch<__half>(const PagedAttnArgs&, int, bool, cudaStream_t);
}  // namespace nexrt

using namespace nexrt;

extern "C" int nexrt_paged_item_cost(void) { return kItemCost; }
extern "C" int nexrt_paged_resident(int dim) { return resident_ctas(dim); }

extern "C" int nexrt_paged_attn(const NexrtPagedAttnArgs* x, void* stream) {
    if (x->size != sizeof(*x)) return cudaErrorInvalidValue;
    if (x->rows < 0 || x->kv_heads < 1 || x->q_heads < 1 || x->q_heads % x->kv_heads || x->width < 0 || x->slots < 1 || x->pages < 0 || x->window < 0 || x->ctas < 1 ||
        x->ctas > kMaxCtas || !(x->softcap >= 0.f))
        return cudaErrorInvalidValue;
    if (x->rows == 0) return 0;
    if (((reinterpret_cast<uintptr_t>(x->k_pages) | reinterpret_cast<uintptr_t>(x->v_pages)) & 15) || x->page % 8 || x->head % 8 || x->slot % 8) return cudaErrorInvalidValue;
    // a row is named by its place in units of 16 bytes: pools of up to 64 GB
    if (x->page < 0 || x->slot < 0 || (x->pages > 0 ? x->pages - 1 : 0) * (x->page / 8) + (x->slots - 1) * (x->slot / 8) >= kNoRow) return cudaErrorInvalidValue;
    PagedAttnArgs a = {};
    a.q = x->q; a.k = x->k_pages; a.v = x->v_pages; a.out = x->out; a.lse = static_cast<float*>(x->lse);
    a.q_b = x->q_row; a.q_h = x->q_head; a.o_b = x->out_row; a.o_h = x->out_head; a.head_s = x->head; a.lse_b = x->lse_row;
    a.page_s = static_cast<uint32_t>(x->page / 8); a.slot_s = static_cast<uint32_t>(x->slot / 8);
    a.table = {static_cast<const int*>(x->table), x->table_row, x->rows, x->width, x->slots, x->pages};
    a.lens = static_cast<const int*>(x->lens); a.slopes = static_cast<const float*>(x->slopes);
    a.cuts = static_cast<int4*>(x->scratch);
    a.ws_o = reinterpret_cast<float*>(a.cuts + x->ctas); a.ws_ml = a.ws_o + static_cast<int64_t>(2) * x->ctas * kPaRows * x->dim;
    a.status = static_cast<int*>(x->status);
    a.seqs = x->rows; a.kv_heads = x->kv_heads; a.group = x->q_heads / x->kv_heads; a.head_groups = (a.group + kPaRows - 1) / kPaRows;
    a.by_item = static_cast<int64_t>(x->rows) * x->kv_heads * a.head_groups <= x->ctas;
    a.window = x->window; a.grid = x->ctas; a.scale = x->scale; a.softcap = x->softcap;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // with room for one chunk an item is never cut
    const bool join = static_cast<int64_t>(x->width) * x->slots > kChunk;
    if (x->type == 0) return paged_dispatch<__nv_bfloat16>(a, x->dim, join, st);
    return x->type == 1 ? paged_dispatch<__half>(a, x->dim, join, st) : static_cast<int>(cudaErrorInvalidValue);
}

// Host forms of the index arithmetic above, for tests without a GPU.
extern "C" int64_t nexrt_paged_slot(const int* table, int64_t stride, int rows, int width, int page, int pages, int row, int pos) {
    const int p = pos < 0 ? -1 : page_at({table, stride, rows, width, page, pages}, row, pos / page);
    return p < 0 ? -1 : static_cast<int64_t>(p) * page + pos % page;
}
// out [parts][5]: CTA, sequence, item, first chunk, chunks - the walk of every CTA; returns the number of parts (at most `most` are written).
extern "C" int nexrt_paged_split(const int* lens, int seqs, int items, int64_t room, int window, int grid, int64_t* out, int most) {
    int64_t total = 0;
    auto chunks = [&](int b) {
        int lo, hi;
        key_span(lens[b], room, window, lo, hi);
        return chunks_of(lo, hi);
    };
    for (int b = 0; b < seqs; ++b) total += static_cast<int64_t>(cost_of(chunks(b))) * items;
    const int n = active_ctas(total, grid);
    int parts = 0;
    for (int c = 0; total > 0 && c < n; ++c) {
        int64_t x = range_begin(total, c, n), first = 0;
        const int64_t end = range_begin(total, c + 1, n);
        int b = 0;
        while (x < end) {
            const int per = chunks(b), cost = cost_of(per);
            if (x >= first + static_cast<int64_t>(cost) * items) {
                first += static_cast<int64_t>(cost) * items;
                ++b;
                continue;
            }
            const int64_t item = (x - first) / cost, item0 = first + item * cost;
            int c0, c1;
            item_part(item0, per, x, end, c0, c1);
            x = item0 + cost;
            if (c1 <= c0) continue;
            // what the joining kernel expects: the first part with the owner of the first chunk, the last with that of the last
            const bool ends = (c0 != 0 || owner_of(item0 + kItemCost, total, n) == c) && (c1 != per || owner_of(item0 + cost - 1, total, n) == c);
            if (parts < most) {
                int64_t* o = out + static_cast<int64_t>(parts) * 5;
                o[0] = c; o[1] = b; o[2] = item; o[3] = c0; o[4] = ends ? c1 - c0 : -1;
            }
            ++parts;
        }
    }
    return parts;
}
