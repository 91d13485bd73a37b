// paged.cpp -- extern "C" entries of batched attention serving (declared in
// include/nmi_fp8_linear.h): handing out the pages of a KV cache, appending to it, decode attention over it,
// whole or by selected pages, and attention over packed prompts.  The reference serves one sequence from contiguous
// caches and has none of them.
//
// What the host can see is checked here before anything is launched; page tables, lengths and offsets
// are device data, which the kernels keep within bounds (nmi_paged.hpp) and report afterwards
// (NMI_ERR_ASYNC).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "nmi_fp8_linear.h"
#include "nmi_launch.hpp"

using namespace nmi;

namespace {

int refuse(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int refuse(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    set_last_error("%s", buf);
    return code;
}

int hip_status(hipError_t e, const char* what) {
    if (e == hipSuccess) return NMI_OK;
    return refuse((int)e, "%s: %s (hipError %d)", what, hipGetErrorString(e), (int)e);
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Rows of `heads` head vectors: base 16-byte aligned, row stride a multiple of 8 elements (and small
// enough for the 32-bit offsets that the kernels add to a tile's address).
constexpr int64_t kMaxStride = 1 << 24;
bool rows_ok(const void* p, int64_t ld, int heads) {
    return ld >= (int64_t)heads * kPagedHead && ld <= kMaxStride && ld % 8 == 0 && aligned(p, 16);
}

// Workgroups along one axis of a launch, of 256 threads each: the axis has less than 2^32 threads.
constexpr int64_t kMaxGroups256 = (1 << 24) - 1;
constexpr int64_t kMaxGroups1024 = (1 << 22) - 1;       // of 1024 threads each

// A cache descriptor as the kernels take it; 0 or an NMI_ERR_* with the message set.
int check_cache(const char* fn, const nmi_paged_kv* c, PagedKv* out, BlockScales* blocks) {
    if (!c) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL cache", fn);
    if (!c->k_pages || !c->v_pages || !c->page_table)
        return refuse(NMI_ERR_INVALID_ARG, "%s: NULL pages or page table", fn);
    if (c->kv_type != NMI_KV_BF16 && c->kv_type != NMI_KV_E4M3 && c->kv_type != NMI_KV_E4M3_BLOCK)
        return refuse(NMI_ERR_INVALID_ARG, "%s: kv_type=%d is none of NMI_KV_BF16, NMI_KV_E4M3 and NMI_KV_E4M3_BLOCK", fn,
                      c->kv_type);
    if (c->page_size < kPagedMinPage || c->page_size > kPagedMaxPage || (c->page_size & (c->page_size - 1)) != 0)
        return refuse(NMI_ERR_INVALID_ARG, "%s: page_size=%d (need a power of two from %d to %d)", fn, c->page_size,
                      kPagedMinPage, kPagedMaxPage);
    if (c->n_pages < 1 || c->max_pages < 1 || c->n_kv_heads < 1 || c->page_table_stride < c->max_pages ||
        (int64_t)c->max_pages * c->page_size > kPagedMaxPositions)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: n_pages=%d max_pages=%d page_table_stride=%lld n_kv_heads=%d page_size=%d (need all >= 1, "
                      "page_table_stride >= max_pages, at most 2^30 positions per sequence)",
                      fn, c->n_pages, c->max_pages, (long long)c->page_table_stride, c->n_kv_heads, c->page_size);
    const int e4m3 = c->kv_type != NMI_KV_BF16, block = c->kv_type == NMI_KV_E4M3_BLOCK, per16 = e4m3 ? 16 : 8, size = e4m3 ? 1 : 2;
    if (c->token_stride < kPagedHead || c->head_stride < kPagedHead || c->page_stride < kPagedHead ||
        c->token_stride > kMaxStride)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: page_stride=%lld head_stride=%lld token_stride=%lld (need at least the %d dims of a head, "
                      "token_stride at most 2^24)",
                      fn, (long long)c->page_stride, (long long)c->head_stride, (long long)c->token_stride, kPagedHead);
    if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || c->page_stride % per16 || c->head_stride % per16 ||
        c->token_stride % per16 || !aligned(c->page_table, 4) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return refuse(NMI_ERR_ALIGNMENT,
                      "%s: pages and their strides must be multiples of 16 bytes, the page table and the scales 4-byte "
                      "aligned",
                      fn);
    if (!e4m3 && (c->k_scale || c->v_scale))
        return refuse(NMI_ERR_INVALID_ARG, "%s: a bf16 cache takes no scales", fn);
    if (block && (!c->k_scale || !c->v_scale))
        return refuse(NMI_ERR_INVALID_ARG, "%s: a cache with scales of blocks needs both", fn);
    *out = PagedKv{static_cast<uint8_t*>(c->k_pages), static_cast<uint8_t*>(c->v_pages), c->page_stride * size,
                   c->head_stride * size, c->token_stride * size, c->page_table, c->page_table_stride,
                   block ? nullptr : c->k_scale, block ? nullptr : c->v_scale, c->n_pages, c->max_pages,
                   __builtin_ctz((unsigned)c->page_size), c->n_kv_heads, nullptr};
    if (block) *blocks = BlockScales{const_cast<float*>(c->k_scale), const_cast<float*>(c->v_scale)};
    return NMI_OK;
}

KvForm form_of(const nmi_paged_kv* c) {
    return c->kv_type == NMI_KV_BF16 ? KvForm::Bf16 : c->kv_type == NMI_KV_E4M3 ? KvForm::E4m3 : KvForm::Block;
}

// The arguments that the decode entries share, checked, as the kernels take them; 0 or an NMI_ERR_*.
int check_decode(const char* fn, const nmi_paged_kv* cache, const void* q_bf16, int64_t ldq, void* o_bf16, int64_t ldo,
                 const int32_t* kv_lens, int batch, int n_heads, float scale, PagedDecodeArgs* out) {
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    PagedDecodeArgs& a = *out;
    if (const int rc = check_cache(fn, cache, &a.kv, &a.blocks)) return rc;
    if (!q_bf16 || !o_bf16 || !kv_lens) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL q, o or kv_lens", fn);
    const int n_kv = a.kv.n_kv;
    if (batch < 1 || n_heads < n_kv || n_heads % n_kv || n_heads > 65535)
        return refuse(NMI_ERR_INVALID_ARG, "%s: batch=%d n_heads=%d n_kv_heads=%d (need batch >= 1, n_heads a multiple)",
                      fn, batch, n_heads, n_kv);
    // the joining launch's axis; and every sequence at its longest, in tiles, summed by the kernel in 32 bits
    if (batch > kMaxGroups256)
        return refuse(NMI_ERR_INVALID_ARG, "%s: batch=%d is too large for one launch", fn, batch);
    if ((int64_t)batch * (((int64_t)a.kv.max_pages << a.kv.page_shift) / kPagedTile) > INT32_MAX)
        return refuse(NMI_ERR_INVALID_ARG, "%s: batch=%d sequences of up to %lld positions are more than 2^35", fn, batch,
                      (long long)a.kv.max_pages << a.kv.page_shift);
    if (!(scale > 0.f) || !std::isfinite(scale))
        return refuse(NMI_ERR_INVALID_ARG, "%s: scale=%g must be positive and finite", fn, (double)scale);
    if (!rows_ok(q_bf16, ldq, n_heads) || ldo < (int64_t)n_heads * kPagedHead || ldo % 2 || !aligned(o_bf16, 4) ||
        !aligned(kv_lens, 4))
        return refuse(NMI_ERR_ALIGNMENT,
                      "%s: q must be 16-byte aligned with a row stride of at least its heads' columns, a multiple of "
                      "8 elements and at most 2^24; o 4-byte aligned with an even one; kv_lens 4-byte aligned (ldq=%lld ldo=%lld)",
                      fn, (long long)ldq, (long long)ldo);
    a.q = static_cast<const uint16_t*>(q_bf16);
    a.o = static_cast<uint16_t*>(o_bf16);
    a.ldq = ldq;
    a.ldo = ldo;
    a.lens = kv_lens;
    a.batch = batch;
    a.H = n_heads;
    a.group = n_heads / n_kv;
    a.scale2 = 1.4426950408889634f * scale;
    return NMI_OK;
}

// Whether the decode's sequences are short enough for a workgroup each (by what the table's rows can hold).
bool whole_rows(const PagedDecodeArgs& a) {
    return sdpa_decode_paged_whole((int64_t)a.kv.max_pages << a.kv.page_shift, a.batch, a.kv.n_kv, a.group);
}

// A workspace given, checked, or one from the bump allocator.
int take_workspace(const char* fn, size_t need, void** workspace, size_t bytes) {
    if (!*workspace) return nmi_alloc(need, workspace);
    if (!aligned(*workspace, 16)) return refuse(NMI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
    if (bytes < need) return refuse(NMI_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, bytes, need);
    return NMI_OK;
}

struct SparseLayout {
    size_t scores, rows, lens, decode, total;       // byte offsets; scores, rows and lens only where pages are chosen
};
SparseLayout sparse_layout(int batch, int n_heads, int n_kv, int max_pages, int n_select) {
    const size_t groups = (size_t)batch * n_kv, some = n_select >= max_pages ? 0 : 1;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    SparseLayout w{};
    w.rows = up(some * groups * max_pages * sizeof(float));
    w.lens = w.rows + up(some * groups * n_select * sizeof(int32_t));
    w.decode = w.lens + up(some * batch * sizeof(int32_t));
    w.total = w.decode + sdpa_decode_paged_workspace_bytes(batch, n_heads, n_kv);
    return w;
}

}  // namespace

extern "C" {

int nmi_kv_append_paged(const nmi_paged_kv* cache, const void* q_bf16, int64_t ldq, const void* k_bf16, int64_t ldk,
                        const void* v_bf16, int64_t ldv, void* q_out_bf16, int64_t ldqo, void* k_out_bf16, int64_t ldko,
                        const int32_t* cu_seqlens, const int32_t* start_pos, int batch, int tokens, int n_heads,
                        const float* inv_freq, int rotary_dim, int interleaved, void* stream) {
    const char* fn = "nmi_kv_append_paged";
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    AppendArgs a{};
    if (const int rc = check_cache(fn, cache, &a.kv, &a.blocks)) return rc;
    if (!k_bf16 || !v_bf16 || !start_pos) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL k, v or start_pos", fn);
    if (batch < 1 || tokens < 1 || tokens > kMaxGroups256 || (!cu_seqlens && tokens != batch))
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: batch=%d tokens=%d (need both >= 1, less than 2^24 tokens, and as many as sequences where "
                      "cu_seqlens is NULL)",
                      fn, batch, tokens);
    if (rotary_dim < 0 || rotary_dim > kPagedHead || rotary_dim % 16 || (rotary_dim > 0) != (inv_freq != nullptr))
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: rotary_dim=%d (need a multiple of 16 up to %d, with inv_freq, or 0 without)", fn, rotary_dim,
                      kPagedHead);
    if ((q_bf16 != nullptr) != (q_out_bf16 != nullptr) || ((q_bf16 || k_out_bf16) && !rotary_dim))
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: q and q_out go together, and they and k_out only with a rotation", fn);
    const int n_kv = a.kv.n_kv;
    if (q_bf16 && (n_heads < 1 || n_heads % n_kv))
        return refuse(NMI_ERR_INVALID_ARG, "%s: n_heads=%d n_kv_heads=%d (need a multiple)", fn, n_heads, n_kv);
    if (!rows_ok(k_bf16, ldk, n_kv) || !rows_ok(v_bf16, ldv, n_kv) || (q_bf16 && !rows_ok(q_bf16, ldq, n_heads)) ||
        (q_bf16 && !rows_ok(q_out_bf16, ldqo, n_heads)) || (k_out_bf16 && !rows_ok(k_out_bf16, ldko, n_kv)))
        return refuse(NMI_ERR_ALIGNMENT,
                      "%s: q, k, v and the outputs must be 16-byte aligned with row strides of at least their heads' "
                      "columns, multiples of 8 elements and at most 2^24 (ldq=%lld ldk=%lld ldv=%lld ldqo=%lld ldko=%lld)",
                      fn, (long long)ldq, (long long)ldk, (long long)ldv, (long long)ldqo, (long long)ldko);
    if (!aligned(cu_seqlens, 4) || !aligned(start_pos, 4) || !aligned(inv_freq, 4))
        return refuse(NMI_ERR_ALIGNMENT, "%s: cu_seqlens, start_pos and inv_freq must be 4-byte aligned", fn);
    a.q = static_cast<const uint16_t*>(q_bf16);
    a.k = static_cast<const uint16_t*>(k_bf16);
    a.v = static_cast<const uint16_t*>(v_bf16);
    a.q_out = static_cast<uint16_t*>(q_out_bf16);
    a.k_out = static_cast<uint16_t*>(k_out_bf16);
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldqo = ldqo;
    a.ldko = ldko;
    a.cu = cu_seqlens;
    a.start = start_pos;
    a.inv_freq = inv_freq;
    a.batch = batch;
    a.tokens = tokens;
    a.H = n_heads;
    a.rotary = rotary_dim;
    a.interleaved = interleaved != 0;
    a.kv.error = async_error_word(AsyncKind::Paged);
    if (form_of(cache) == KvForm::Block) {
        if (cu_seqlens && most_blocks(tokens, batch) >= kMaxGroups256)
            return refuse(NMI_ERR_INVALID_ARG, "%s: batch=%d tokens=%d are too many blocks", fn, batch, tokens);
        return hip_status(launch_kv_append_block(a, static_cast<hipStream_t>(stream)), fn);
    }
    return hip_status(launch_kv_append(a, cache->kv_type == NMI_KV_E4M3, static_cast<hipStream_t>(stream)), fn);
}

int nmi_kv_assign_paged(const int32_t* lens, const int32_t* new_lens, int32_t* page_table, int64_t page_table_stride,
                        int max_pages, int page_size, int32_t* free_pages, const int32_t* free_count, int n_pages, int batch,
                        int tokens, int32_t* start_pos, int32_t* kv_lens, int32_t* cu_seqlens, int64_t* slots,
                        int32_t* lens_out, int32_t* free_count_out, void* stream) {
    const char* fn = "nmi_kv_assign_paged";
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    if (!lens || !page_table || !free_pages || !free_count || !start_pos || !kv_lens || !slots || !lens_out || !free_count_out)
        return refuse(NMI_ERR_INVALID_ARG, "%s: NULL pointer argument", fn);
    if (page_size < kPagedMinPage || page_size > kPagedMaxPage || (page_size & (page_size - 1)) != 0)
        return refuse(NMI_ERR_INVALID_ARG, "%s: page_size=%d (need a power of two from %d to %d)", fn, page_size,
                      kPagedMinPage, kPagedMaxPage);
    if (n_pages < 1 || max_pages < 1 || page_table_stride < max_pages ||
        (int64_t)max_pages * page_size > kPagedMaxPositions)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: n_pages=%d max_pages=%d page_table_stride=%lld page_size=%d (need all >= 1, page_table_stride >= "
                      "max_pages, at most 2^30 positions per sequence)",
                      fn, n_pages, max_pages, (long long)page_table_stride, page_size);
    if (batch < 1 || batch > kMaxGroups256 || tokens < 0 || tokens > kMaxGroups256 || (!cu_seqlens && tokens != batch))
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: batch=%d tokens=%d (need batch >= 1, tokens >= 0, both less than 2^24, and as many tokens as "
                      "sequences where cu_seqlens is NULL)",
                      fn, batch, tokens);
    if (!aligned(lens, 4) || !aligned(new_lens, 4) || !aligned(page_table, 4) || !aligned(free_pages, 4) ||
        !aligned(free_count, 4) || !aligned(start_pos, 4) || !aligned(kv_lens, 4) || !aligned(cu_seqlens, 4) ||
        !aligned(slots, 8) || !aligned(lens_out, 4) || !aligned(free_count_out, 4))
        return refuse(NMI_ERR_ALIGNMENT, "%s: slots must be 8-byte aligned, all else 4-byte", fn);
    AssignArgs a{};
    a.lens = lens;
    a.add = new_lens;
    a.table = page_table;
    a.table_stride = page_table_stride;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.start = start_pos;
    a.kv_lens = kv_lens;
    a.cu = cu_seqlens;
    a.lens_out = lens_out;
    a.free_count_out = free_count_out;
    a.slots = slots;
    a.n_pages = n_pages;
    a.max_pages = max_pages;
    a.page_shift = __builtin_ctz((unsigned)page_size);
    a.batch = batch;
    a.tokens = tokens;
    a.error = async_error_word(AsyncKind::Paged);
    return hip_status(launch_kv_assign(a, static_cast<hipStream_t>(stream)), fn);
}

int nmi_kv_bounds_paged(const nmi_paged_kv* cache, void* k_bounds_bf16, const int32_t* cu_seqlens, const int32_t* start_pos,
                        int batch, int tokens, void* stream) {
    const char* fn = "nmi_kv_bounds_paged";
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    BoundsArgs a{};
    if (const int rc = check_cache(fn, cache, &a.kv, &a.blocks)) return rc;
    if (!k_bounds_bf16 || !start_pos) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL k_bounds or start_pos", fn);
    if (batch < 1 || tokens < 1 || (!cu_seqlens && tokens != batch) || batch > kMaxGroups256 || tokens > kMaxGroups256 ||
        most_pages_completed(tokens, batch, a.kv.page_shift) >= kMaxGroups256 || a.kv.n_kv > 65535)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: batch=%d tokens=%d n_kv_heads=%d (need all >= 1, less than 2^24 tokens and pages, at most 65535 "
                      "heads, and as many tokens as sequences where cu_seqlens is NULL)",
                      fn, batch, tokens, a.kv.n_kv);
    if (!aligned(k_bounds_bf16, 16) || !aligned(cu_seqlens, 4) || !aligned(start_pos, 4))
        return refuse(NMI_ERR_ALIGNMENT, "%s: k_bounds must be 16-byte aligned, cu_seqlens and start_pos 4-byte", fn);
    a.bounds = static_cast<uint16_t*>(k_bounds_bf16);
    a.cu = cu_seqlens;
    a.start = start_pos;
    a.batch = batch;
    a.tokens = tokens;
    a.kv.error = async_error_word(AsyncKind::Paged);
    return hip_status(launch_kv_bounds(a, form_of(cache), static_cast<hipStream_t>(stream)), fn);
}

size_t nmi_sdpa_decode_paged_workspace_bytes(int batch, int n_heads, int n_kv_heads) {
    if (batch < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads) return 0;
    return sdpa_decode_paged_workspace_bytes(batch, n_heads, n_kv_heads);
}

int nmi_sdpa_decode_paged(const nmi_paged_kv* cache, const void* q_bf16, int64_t ldq, void* o_bf16, int64_t ldo,
                          const int32_t* kv_lens, int batch, int n_heads, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* fn = "nmi_sdpa_decode_paged";
    PagedDecodeArgs a{};
    if (const int rc = check_decode(fn, cache, q_bf16, ldq, o_bf16, ldo, kv_lens, batch, n_heads, scale, &a)) return rc;
    const size_t need = sdpa_decode_paged_workspace_bytes(batch, n_heads, a.kv.n_kv);
    if (const int rc = take_workspace(fn, need, &workspace, workspace_bytes)) return rc;
    a.kv.error = async_error_word(AsyncKind::Paged);
    const KvForm form = form_of(cache);
    // (the older forms keep the order of their sums)
    return hip_status(launch_sdpa_decode_paged(a, form, form == KvForm::Block && whole_rows(a), workspace, static_cast<hipStream_t>(stream)),
                      fn);
}

size_t nmi_sdpa_decode_paged_sparse_workspace_bytes(int batch, int n_heads, int n_kv_heads, int max_pages, int n_select) {
    if (batch < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads || max_pages < 1 || n_select < 1) return 0;
    return sparse_layout(batch, n_heads, n_kv_heads, max_pages, n_select).total;
}

int nmi_sdpa_decode_paged_sparse(const nmi_paged_kv* cache, const void* q_bf16, int64_t ldq, void* o_bf16, int64_t ldo,
                                 const int32_t* kv_lens, const void* k_bounds_bf16, int n_select, int32_t* selected, int batch,
                                 int n_heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "nmi_sdpa_decode_paged_sparse";
    PagedDecodeArgs a{};
    if (const int rc = check_decode(fn, cache, q_bf16, ldq, o_bf16, ldo, kv_lens, batch, n_heads, scale, &a)) return rc;
    if (!k_bounds_bf16) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL k_bounds", fn);
    if (n_select < 1) return refuse(NMI_ERR_INVALID_ARG, "%s: n_select=%d (need at least the newest page)", fn, n_select);
    if ((int64_t)batch * a.kv.n_kv > kMaxGroups1024)
        return refuse(NMI_ERR_INVALID_ARG, "%s: batch=%d n_kv_heads=%d are too many for one launch", fn, batch, a.kv.n_kv);
    if (!aligned(k_bounds_bf16, 16) || !aligned(selected, 4))
        return refuse(NMI_ERR_ALIGNMENT, "%s: k_bounds must be 16-byte aligned, selected 4-byte", fn);
    const SparseLayout w = sparse_layout(batch, n_heads, a.kv.n_kv, a.kv.max_pages, n_select);
    if (const int rc = take_workspace(fn, w.total, &workspace, workspace_bytes)) return rc;
    char* base = static_cast<char*>(workspace);
    const bool all = n_select >= a.kv.max_pages;        // no sequence has more pages than that
    SelectArgs s{};
    s.kv = a.kv;
    s.q = a.q;
    s.ldq = ldq;
    s.lens = kv_lens;
    s.bounds = static_cast<const uint16_t*>(k_bounds_bf16);
    s.selected = selected;
    s.batch = batch;
    s.group = a.group;
    s.select = n_select;
    if (!all) {
        s.scores = reinterpret_cast<float*>(base + w.scores);
        s.rows = reinterpret_cast<int32_t*>(base + w.rows);
        s.out_lens = reinterpret_cast<int32_t*>(base + w.lens);
        a.kv.page_table = s.rows;
        a.kv.table_stride = (int64_t)a.kv.n_kv * n_select;
        a.table_head_stride = n_select;
        a.kv.max_pages = n_select;
        a.lens = s.out_lens;
    }
    if (!all || selected)
        if (const int rc = hip_status(launch_page_select(s, static_cast<hipStream_t>(stream)), fn)) return rc;
    a.kv.error = async_error_word(AsyncKind::Paged);
    return hip_status(
        launch_sdpa_decode_paged(a, form_of(cache), whole_rows(a), base + w.decode, static_cast<hipStream_t>(stream)), fn);
}

int nmi_sdpa_prefill_packed_bf16(const void* q_bf16, int64_t ldq, const void* k_bf16, int64_t ldk, const void* v_bf16,
                                 int64_t ldv, void* o_bf16, int64_t ldo, const int32_t* cu_seqlens, int batch, int tokens,
                                 int n_heads, int n_kv_heads, float scale, void* stream) {
    const char* fn = "nmi_sdpa_prefill_packed_bf16";
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    if (!q_bf16 || !k_bf16 || !v_bf16 || !o_bf16 || !cu_seqlens)
        return refuse(NMI_ERR_INVALID_ARG, "%s: NULL pointer argument", fn);
    if (batch < 1 || tokens < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: batch=%d tokens=%d n_heads=%d n_kv_heads=%d (need all >= 1, n_heads a multiple of n_kv_heads)",
                      fn, batch, tokens, n_heads, n_kv_heads);
    if (tokens > kPagedMaxPositions || sdpa_prefill_packed_tiles(tokens, batch) * n_heads > kMaxGroups256)
        return refuse(NMI_ERR_INVALID_ARG, "%s: tokens=%d batch=%d n_heads=%d are too many query tiles", fn, tokens, batch,
                      n_heads);
    if (!(scale > 0.f) || !std::isfinite(scale))
        return refuse(NMI_ERR_INVALID_ARG, "%s: scale=%g must be positive and finite", fn, (double)scale);
    if (!rows_ok(q_bf16, ldq, n_heads) || !rows_ok(k_bf16, ldk, n_kv_heads) || !rows_ok(v_bf16, ldv, n_kv_heads) ||
        ldo < (int64_t)n_heads * kPagedHead || ldo % 4 || !aligned(o_bf16, 8) || !aligned(cu_seqlens, 4))
        return refuse(NMI_ERR_ALIGNMENT,
                      "%s: q, k, v must be 16-byte aligned with row strides of at least their heads' columns, multiples "
                      "of 8 elements and at most 2^24; o 8-byte aligned with a multiple of 4; cu_seqlens 4-byte aligned (ldq=%lld "
                      "ldk=%lld ldv=%lld ldo=%lld)",
                      fn, (long long)ldq, (long long)ldk, (long long)ldv, (long long)ldo);
    return hip_status(launch_sdpa_prefill_packed(static_cast<const uint16_t*>(q_bf16), ldq,
                                                 static_cast<const uint16_t*>(k_bf16), ldk,
                                                 static_cast<const uint16_t*>(v_bf16), ldv, static_cast<uint16_t*>(o_bf16),
                                                 ldo, cu_seqlens, batch, tokens, n_heads, n_kv_heads, scale,
                                                 static_cast<hipStream_t>(stream)),
                      fn);
}

}  // extern "C"
