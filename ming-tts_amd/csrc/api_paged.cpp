// The C ABI of the operators on caches in pages and on windows with first positions that stay visible
// (include/mingtts_hip.h): argument validation, before any HIP call, and the launchers' operands.
#include "api_checks.hpp"
#include "mingtts_hip.h"
#include "mt_internal.hpp"

namespace mt {

namespace {

int validate_paged(const char *who, const mt_paged_kv *c, uint32_t B, uint32_t hkv, PagedArgs &out) {
    if (!c) return set_error(MT_EINVAL, "%s: null kv", who);
    if (c->cache_t != DT_F32 && c->cache_t != DT_F16 && c->cache_t != DT_F8)
        return set_error(MT_EINVAL, "%s: kv must be f32, f16 or f8", who);
    if (!c->k || !c->v || !c->table) return set_error(MT_EINVAL, "%s: null k, v or table of kv", who);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->table, 4))
        return set_error(MT_EINVAL, "%s: k and v of kv must be 16-byte, its table 4-byte aligned", who);
    if (c->pages == 0) return set_error(MT_EINVAL, "%s: kv has no pages", who);
    if (c->page_len == 0 || c->page_len % 16 || c->page_len > 32768)
        return set_error(MT_EINVAL, "%s: page_len %u is no multiple of 16 up to 32768", who, c->page_len);
    const uint64_t slots = static_cast<uint64_t>(c->table_len) * c->page_len;
    if (slots == 0 || slots > (1u << 30))
        return set_error(MT_EINVAL, "%s: %u entries of %u slots are outside 1..2^30 slots", who, c->table_len, c->page_len);
    if (B > 1 && c->table_stride < c->table_len)
        return set_error(MT_EINVAL, "%s: table_stride %u < table_len %u", who, c->table_stride, c->table_len);
    const uint64_t rows = static_cast<uint64_t>(hkv) * c->page_len;
    const uint64_t most = (1ull << 48) / c->pages;  // elements of a page at which the pool's bytes fit 64 bits
    if (c->stride < rows * 64 || c->stride % 16 || c->stride > most)
        return set_error(MT_EINVAL, "%s: stride of kv smaller than one page, no multiple of 16 or too large", who);
    if (c->cache_t == DT_F8) {
        if (!c->k_scale || !c->v_scale) return set_error(MT_EINVAL, "%s: null scales of kv", who);
        if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
            return set_error(MT_EINVAL, "%s: scales of kv must be 4-byte aligned", who);
        if (c->scale_stride < rows || c->scale_stride % 4 || c->scale_stride > most)
            return set_error(MT_EINVAL, "%s: scale_stride of kv smaller than one page, no multiple of 4 or too large", who);
    }
    out = PagedArgs{c->k, c->v, c->k_scale, c->v_scale, c->stride, c->scale_stride, c->table, c->pages, c->page_len,
                    static_cast<uint32_t>(slots), B > 1 ? c->table_stride : 0, (1ull << 37) / (c->page_len / 16) + 1};
    return MT_OK;
}

// The memory of the pools and of the table.
struct PagedRuns {
    Runs r[5];
    PagedRuns(const PagedArgs &c, int ct, uint32_t B, uint32_t hkv) {
        const uint64_t rows = static_cast<uint64_t>(hkv) * c.page_len, es = elem_bytes(ct), scales = ct == DT_F8 ? rows : 0;
        r[0] = Runs{c.k, rows * 64 * es, c.stride * es, c.pages};
        r[1] = Runs{c.v, rows * 64 * es, c.stride * es, c.pages};
        r[2] = Runs{c.ks, scales, c.sstride, c.pages};
        r[3] = Runs{c.vs, scales, c.sstride, c.pages};
        r[4] = Runs{c.table, span(B, c.len / c.page_len, c.table_stride, 4), 0, 1};
    }
    bool meet_each_other() const {
        for (int i = 1; i < 5; i++)
            for (int j = 0; j < i; j++)
                if (meet(r[i], r[j])) return true;
        return false;
    }
};

// The workspace of a plan: its parts' sums, references and weights' sums, and their flags.
uint64_t window_bytes(const WindowPlan &p, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv) {
    if (p.parts <= 1) return 0;
    const uint64_t rows = static_cast<uint64_t>(T) * (hq / hkv), tiles = static_cast<uint64_t>(B) * hkv * ((rows + 15) / 16);
    return (static_cast<uint64_t>(B) * T * hq * 33 + tiles) * p.parts * 8;
}

// What mt_attention_paged and mt_attention_sinks check alike, behind their caches: `a` has those, `caches` their memory.
int attend(const char *who, WindowArgs &a, int ct, const Runs *caches, int n_caches, const float *q, uint32_t ldq, uint32_t B, uint32_t T,
           uint32_t hq, uint32_t hkv, const uint32_t *pos, const uint32_t *counts, uint32_t len_max, uint32_t window,
           uint32_t sinks, float *out, uint32_t ldo, float scale, void *workspace, uint64_t workspace_bytes, mt_stream_t stream) {
    if (!q || !out) return set_error(MT_EINVAL, "%s: null pointer", who);
    const uint64_t all = static_cast<uint64_t>(B) * T, w = static_cast<uint64_t>(hq) * 64;
    if (ldq < w || ldo < w) return set_error(MT_EINVAL, "%s: ldq / ldo < hq * 64", who);
    if (!aligned(q, 16) || ldq % 4 || !aligned(out, 16) || ldo % 4)
        return set_error(MT_EINVAL, "%s: q / out must be 16-byte aligned with 16-byte row strides", who);
    const uint64_t ob = span(all, w, ldo, 4);
    if (meet(q, span(all, w, ldq, 4), out, ob)) return set_error(MT_EINVAL, "%s: out overlaps q", who);
    for (int i = 0; i < n_caches; i++)
        if (meet(caches[i].p, caches[i].all(), out, ob)) return set_error(MT_EINVAL, "%s: out overlaps the caches", who);
    const WindowPlan plan = window_plan(B, T, hq, hkv, len_max ? len_max : a.kv.len, window, sinks, ct);
    const uint64_t need = window_bytes(plan, B, T, hq, hkv);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(MT_EINVAL, "%s: needs %llu bytes of 16-byte aligned workspace, got %llu", who,
                         static_cast<unsigned long long>(need), static_cast<unsigned long long>(workspace ? workspace_bytes : 0));
    if (need) {
        bool met = meet(workspace, need, q, span(all, w, ldq, 4)) || meet(workspace, need, out, ob);
        for (int i = 0; i < n_caches; i++) met = met || meet(workspace, need, caches[i].p, caches[i].all());
        if (met) return set_error(MT_EINVAL, "%s: the workspace overlaps q, out or the caches", who);
    }
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.hq = hq;
    a.hkv = hkv;
    a.window = window;
    a.sinks = sinks;
    a.rows = RowsArgs{pos, counts, B, T};
    a.scale = scale;
    a.group = hq / hkv;
    a.group_magic = static_cast<uint32_t>((1ull << 32) / a.group + 1);
    a.part = static_cast<float *>(workspace);
    return launch_attention_window(a, plan, ct, reinterpret_cast<hipStream_t>(stream));
}

int validate_heads(const char *who, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv) {
    const int rc = validate_rows(who, B, T, hq, hkv);
    if (rc) return rc;
    if (hq == 0 || hq % hkv) return set_error(MT_EINVAL, "%s: hq %u must be a positive multiple of hkv %u", who, hq, hkv);
    const uint64_t G = hq / hkv;
    if (G > 4096 || static_cast<uint64_t>(B) * T * G > 0xFFFFFFFFull / G)
        return set_error(MT_EINVAL, "%s: %u x %u rows of %u query heads a key head are too many", who, B, T, hq / hkv);
    return MT_OK;
}

}  // namespace

}  // namespace mt

using namespace mt;

extern "C" {

int mt_rope_append_paged(const float *qkv, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, const uint32_t *pos,
                         const uint32_t *counts, uint32_t offset, const mt_paged_kv *kv, const float *inv_freq, float *q,
                         uint32_t ldo, mt_stream_t stream) {
    const char *who = "mt_rope_append_paged";
    int rc = validate_rows(who, B, T, hq, hkv);
    if (rc) return rc;
    if (B == 0 || T == 0) return MT_OK;
    PagedArgs c;
    rc = validate_paged(who, kv, B, hkv, c);
    if (rc) return rc;
    uint64_t in, outb;
    rc = validate_qkv(who, qkv, ldq, B, T, hq, hkv, inv_freq, q, ldo, in, outb);
    if (rc) return rc;
    const PagedRuns caches(c, kv->cache_t, B, hkv);
    for (const Runs &r : caches.r)
        if (meet(r.p, r.all(), qkv, in) || meet(r.p, r.all(), q, outb))
            return set_error(MT_EINVAL, "%s: the caches overlap qkv or q", who);
    if (caches.meet_each_other()) return set_error(MT_EINVAL, "%s: the caches or the table overlap each other", who);
    return launch_rope_append_paged(qkv, ldq, RowsArgs{pos, counts, B, T}, hq, hkv, offset, c, kv->cache_t, inv_freq, q, ldo,
                                    reinterpret_cast<hipStream_t>(stream));
}

uint64_t mt_attention_window_workspace(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t len_max, uint32_t window,
                                       uint32_t sinks, mt_dtype cache_t) {
    if (validate_heads("mt_attention_window_workspace", B, T, hq, hkv) || B == 0 || T == 0) return 0;
    return window_bytes(window_plan(B, T, hq, hkv, len_max, window, sinks, cache_t), B, T, hq, hkv);
}

int mt_attention_paged(const float *q, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, const uint32_t *pos,
                       const uint32_t *counts, const mt_paged_kv *kv, uint32_t len_max, uint32_t window, uint32_t sinks, float *out,
                       uint32_t ldo, float scale, void *workspace, uint64_t workspace_bytes, mt_stream_t stream) {
    const char *who = "mt_attention_paged";
    int rc = validate_heads(who, B, T, hq, hkv);
    if (rc) return rc;
    if (B == 0 || T == 0) return MT_OK;
    WindowArgs a{};
    rc = validate_paged(who, kv, B, hkv, a.kv);
    if (rc) return rc;
    const PagedRuns caches(a.kv, kv->cache_t, B, hkv);
    return attend(who, a, kv->cache_t, caches.r, 5, q, ldq, B, T, hq, hkv, pos, counts, len_max, window, sinks, out, ldo, scale, workspace,
                  workspace_bytes, stream);
}

int mt_attention_sinks(const float *q, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, const uint32_t *pos,
                       const uint32_t *counts, const mt_kv *kv, uint32_t len_max, uint32_t window, uint32_t sinks, float *out,
                       uint32_t ldo, float scale, void *workspace, uint64_t workspace_bytes, mt_stream_t stream) {
    const char *who = "mt_attention_sinks";
    int rc = validate_heads(who, B, T, hq, hkv);
    if (rc) return rc;
    if (B == 0 || T == 0) return MT_OK;
    KvArgs c;
    rc = validate_kv(who, "kv", kv, B, hkv, c);
    if (rc) return rc;
    WindowArgs a{};
    a.kv = PagedArgs{c.k, c.v, c.ks, c.vs, c.stride, c.sstride, nullptr, 0, c.len, c.len, 0, 0};
    const KvRuns caches(c, kv->cache_t, B, hkv);
    return attend(who, a, kv->cache_t, caches.r, 4, q, ldq, B, T, hq, hkv, pos, counts, len_max, window, sinks, out, ldo, scale, workspace,
                  workspace_bytes, stream);
}

}  // extern "C"
