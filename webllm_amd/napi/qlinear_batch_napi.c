/*
 * Node-API binding of the entry points of a pass over many requests (include/qlinear.h): paged caches, attention of a batch,
 * low-rank adapters. Handles are those of qlinear_napi.node, whose exports are the reference path's and a drafted pass's.
 */
#include "napi_util.h"

typedef struct {
    const char* name;
    int32_t* out;
} int_field;
typedef struct {
    const char* name;
    uint64_t* out;
    int none;                     /* null is QL_NONE */
} off_field;

static int get_fields(napi_env env, napi_value obj, const off_field* offs, size_t n_off, const int_field* ints, size_t n_int)
{
    napi_value v;
    for (size_t i = 0; i < n_off; i++)
        if (prop(env, obj, offs[i].name, &v) || get_u64(env, v, offs[i].out, offs[i].none)) return 1;
    for (size_t i = 0; i < n_int; i++)
        if (prop(env, obj, ints[i].name, &v) || get_i32(env, v, ints[i].out)) return 1;
    return 0;
}

/* {rowStartOff, kvLenOff, pagesOff, nSeq, maxPages, maxRows, maxLen} -> ql_batch_desc */
static int get_batch(napi_env env, napi_value obj, ql_batch_desc* d)
{
    const off_field offs[] = {{"rowStartOff", &d->row_start_off, 0}, {"kvLenOff", &d->kv_len_off, 0}, {"pagesOff", &d->pages_off, 0}};
    const int_field ints[] = {{"nSeq", &d->n_seq}, {"maxPages", &d->max_pages}, {"maxRows", &d->max_rows}, {"maxLen", &d->max_len}};
    return get_fields(env, obj, offs, 3, ints, 4);
}

/* {kOff, vOff, kScaleOff|null, vScaleOff|null, nPage, pageSize, nKvHead, D, cacheDtype} -> ql_paged_desc */
static int get_paged(napi_env env, napi_value obj, ql_paged_desc* d)
{
    const off_field offs[] = {{"kOff", &d->k_off, 0}, {"vOff", &d->v_off, 0}, {"kScaleOff", &d->k_scale_off, 1}, {"vScaleOff", &d->v_scale_off, 1}};
    const int_field ints[] = {{"nPage", &d->n_page}, {"pageSize", &d->page_size}, {"nKvHead", &d->n_kv_head}, {"D", &d->D}, {"cacheDtype", &d->cache_dtype}};
    d->reserved = 0;
    return get_fields(env, obj, offs, 4, ints, 5);
}

/* {aOff, bOff, scaleOff|null, K, N, rank, nAdapter} -> ql_lora_desc */
static int get_lora(napi_env env, napi_value obj, ql_lora_desc* d)
{
    const off_field offs[] = {{"aOff", &d->a_off, 0}, {"bOff", &d->b_off, 0}, {"scaleOff", &d->scale_off, 1}};
    const int_field ints[] = {{"K", &d->K}, {"N", &d->N}, {"rank", &d->rank}, {"nAdapter", &d->n_adapter}};
    return get_fields(env, obj, offs, 3, ints, 4);
}

/* pagedAppend(ctx, rope, weights, act, qOff, kOff, vOff, batch, M, qOutOff, qDtype, cache, paged) */
static napi_value js_paged_append(napi_env env, napi_callback_info info)
{
    napi_value argv[13];
    void *ctx, *w, *act, *cache;
    ql_rope_desc rope;
    ql_batch_desc b;
    ql_paged_desc p;
    uint64_t q, k, v, out;
    int32_t M, dtype;
    if (get_args(env, info, 13, argv) || get_ptr(env, argv[0], &ctx) || get_rope(env, argv[1], &rope) || get_ptr(env, argv[2], &w) ||
        get_ptr(env, argv[3], &act) || get_u64(env, argv[4], &q, 0) || get_u64(env, argv[5], &k, 0) || get_u64(env, argv[6], &v, 0) ||
        get_batch(env, argv[7], &b) || get_i32(env, argv[8], &M) || get_u64(env, argv[9], &out, 0) || get_i32(env, argv[10], &dtype) ||
        get_ptr(env, argv[11], &cache) || get_paged(env, argv[12], &p))
        return NULL;
    throw_rc(env, ql_paged_append((ql_ctx*)ctx, &rope, (ql_arena*)w, (ql_arena*)act, q, k, v, &b, M, out, dtype, (ql_arena*)cache, &p));
    return NULL;
}

/* pagedAttention(ctx, act, qOff, qDtype, cache, paged, batch, M, nHead, outOff) */
static napi_value js_paged_attention(napi_env env, napi_callback_info info)
{
    napi_value argv[10];
    void *ctx, *act, *cache;
    ql_batch_desc b;
    ql_paged_desc p;
    uint64_t q, out;
    int32_t dtype, M, H;
    if (get_args(env, info, 10, argv) || get_ptr(env, argv[0], &ctx) || get_ptr(env, argv[1], &act) || get_u64(env, argv[2], &q, 0) ||
        get_i32(env, argv[3], &dtype) || get_ptr(env, argv[4], &cache) || get_paged(env, argv[5], &p) || get_batch(env, argv[6], &b) ||
        get_i32(env, argv[7], &M) || get_i32(env, argv[8], &H) || get_u64(env, argv[9], &out, 0))
        return NULL;
    throw_rc(env, ql_paged_attention((ql_ctx*)ctx, (ql_arena*)act, q, dtype, (ql_arena*)cache, &p, &b, M, H, out));
    return NULL;
}

/* loraAdd(ctx, adapters[], weights, act, idsOff, xOffs[], xDtype, M, baseOffs[], yOffs[]) */
static napi_value js_lora_add(napi_env env, napi_callback_info info)
{
    napi_value argv[10], e;
    void *ctx, *w, *act;
    ql_lora_desc d[8];
    uint64_t ids, x[8], base[8], y[8];
    uint32_t n;
    int32_t dtype, M;
    if (get_args(env, info, 10, argv) || get_ptr(env, argv[0], &ctx)) return NULL;
    if (napi_get_array_length(env, argv[1], &n) != napi_ok || n == 0 || n > 8) {
        napi_throw_type_error(env, "QL_E_INVALID", "expected an array of 1..8 adapters' descriptors");
        return NULL;
    }
    for (uint32_t i = 0; i < n; i++)
        if (napi_get_element(env, argv[1], i, &e) != napi_ok || get_lora(env, e, &d[i])) return NULL;
    if (get_ptr(env, argv[2], &w) || get_ptr(env, argv[3], &act) || get_u64(env, argv[4], &ids, 0) || get_u64_array(env, argv[5], x, n) ||
        get_i32(env, argv[6], &dtype) || get_i32(env, argv[7], &M) || get_u64_array(env, argv[8], base, n) || get_u64_array(env, argv[9], y, n))
        return NULL;
    throw_rc(env, ql_lora_add((ql_ctx*)ctx, (int32_t)n, d, (ql_arena*)w, (ql_arena*)act, ids, x, dtype, M, base, y));
    return NULL;
}

static napi_value init(napi_env env, napi_value exports)
{
    const napi_property_descriptor fns[] = {
        {"pagedAppend", NULL, js_paged_append, NULL, NULL, NULL, napi_enumerable, NULL},
        {"pagedAttention", NULL, js_paged_attention, NULL, NULL, NULL, napi_enumerable, NULL},
        {"loraAdd", NULL, js_lora_add, NULL, NULL, NULL, napi_enumerable, NULL},
    };
    if (napi_define_properties(env, exports, sizeof fns / sizeof fns[0], fns) != napi_ok) return NULL;
    return exports;
}

NAPI_MODULE(NODE_GYP_MODULE_NAME, init)
