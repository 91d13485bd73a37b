// paged.cpp -- extern "C" entries of batched attention serving (declared in
// include/nmi_fp8_linear.h): appending to a paged KV cache, decode attention over it, and attention
// over packed prompts.  The reference serves one sequence from contiguous caches and has none of them.
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

// A cache descriptor as the kernels take it; 0 or an NMI_ERR_* with the message set.
int check_cache(const char* fn, const nmi_paged_kv* c, PagedKv* out) {
    if (!c) return refuse(NMI_ERR_INVALID_ARG, "%s: NULL cache", fn);
    if (!c->k_pages || !c->v_pages || !c->page_table)
        return refuse(NMI_ERR_INVALID_ARG, "%s: NULL pages or page table", fn);
    if (c->kv_type != NMI_KV_BF16 && c->kv_type != NMI_KV_E4M3)
        return refuse(NMI_ERR_INVALID_ARG, "%s: kv_type=%d is neither NMI_KV_BF16 nor NMI_KV_E4M3", fn, c->kv_type);
    if (c->page_size < kPagedMinPage || c->page_size > kPagedMaxPage || (c->page_size & (c->page_size - 1)) != 0)
        return refuse(NMI_ERR_INVALID_ARG, "%s: page_size=%d (need a power of two from %d to %d)", fn, c->page_size,
                      kPagedMinPage, kPagedMaxPage);
    if (c->n_pages < 1 || c->max_pages < 1 || c->n_kv_heads < 1 || c->page_table_stride < c->max_pages ||
        (int64_t)c->max_pages * c->page_size > kPagedMaxPositions)
        return refuse(NMI_ERR_INVALID_ARG,
                      "%s: n_pages=%d max_pages=%d page_table_stride=%lld n_kv_heads=%d page_size=%d (need all >= 1, "
                      "page_table_stride >= max_pages, at most 2^30 positions per sequence)",
                      fn, c->n_pages, c->max_pages, (long long)c->page_table_stride, c->n_kv_heads, c->page_size);
    const int e4m3 = c->kv_type == NMI_KV_E4M3, per16 = e4m3 ? 16 : 8, size = e4m3 ? 1 : 2;
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
    *out = PagedKv{static_cast<uint8_t*>(c->k_pages), static_cast<uint8_t*>(c->v_pages), c->page_stride * size,
                   c->head_stride * size, c->token_stride * size, c->page_table, c->page_table_stride, c->k_scale,
                   c->v_scale, c->n_pages, c->max_pages, __builtin_ctz((unsigned)c->page_size), c->n_kv_heads, nullptr};
    return NMI_OK;
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
    if (const int rc = check_cache(fn, cache, &a.kv)) return rc;
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
    return hip_status(launch_kv_append(a, cache->kv_type == NMI_KV_E4M3, static_cast<hipStream_t>(stream)), fn);
}

size_t nmi_sdpa_decode_paged_workspace_bytes(int batch, int n_heads, int n_kv_heads) {
    if (batch < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads) return 0;
    return sdpa_decode_paged_workspace_bytes(batch, n_heads, n_kv_heads);
}

int nmi_sdpa_decode_paged(const nmi_paged_kv* cache, const void* q_bf16, int64_t ldq, void* o_bf16, int64_t ldo,
                          const int32_t* kv_lens, int batch, int n_heads, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* fn = "nmi_sdpa_decode_paged";
    if (take_async_error(fn, AsyncKind::Paged)) return NMI_ERR_ASYNC;
    PagedDecodeArgs a{};
    if (const int rc = check_cache(fn, cache, &a.kv)) return rc;
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
    const size_t need = sdpa_decode_paged_workspace_bytes(batch, n_heads, n_kv);
    if (workspace) {
        if (!aligned(workspace, 16)) return refuse(NMI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
        if (workspace_bytes < need)
            return refuse(NMI_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, need);
    } else if (const int rc = nmi_alloc(need, &workspace)) {
        return rc;
    }
    a.q = static_cast<const uint16_t*>(q_bf16);
    a.o = static_cast<uint16_t*>(o_bf16);
    a.ldq = ldq;
    a.ldo = ldo;
    a.lens = kv_lens;
    a.batch = batch;
    a.H = n_heads;
    a.group = n_heads / n_kv;
    a.scale2 = 1.4426950408889634f * scale;
    a.kv.error = async_error_word(AsyncKind::Paged);
    return hip_status(launch_sdpa_decode_paged(a, cache->kv_type == NMI_KV_E4M3, workspace, static_cast<hipStream_t>(stream)),
                      fn);
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
