/* Arguments and errors of the Node-API bindings (qlinear_napi.c, qlinear_batch_napi.c). */
#pragma once
#define NAPI_VERSION 6
#include <node_api.h>

#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/qlinear.h"

#define CHECK_NAPI(env, call)                                             \
    do {                                                                  \
        if ((call) != napi_ok) {                                          \
            napi_throw_error((env), "QL_E_NAPI", "Node-API call failed: " #call); \
            return NULL;                                                  \
        }                                                                 \
    } while (0)

static inline const char* code_name(int rc)
{
    switch (rc) {
    case QL_E_BITS: return "QL_E_BITS";
    case QL_E_GROUP: return "QL_E_GROUP";
    case QL_E_DIMS: return "QL_E_DIMS";
    case QL_E_QWEIGHT_SHORT: return "QL_E_QWEIGHT_SHORT";
    case QL_E_SCALES_SHORT: return "QL_E_SCALES_SHORT";
    case QL_E_QZEROS_SHORT: return "QL_E_QZEROS_SHORT";
    case QL_E_GROUP_PACK: return "QL_E_GROUP_PACK";
    case QL_E_INVALID: return "QL_E_INVALID";
    case QL_E_RANGE: return "QL_E_RANGE";
    case QL_E_ALIGN: return "QL_E_ALIGN";
    case QL_E_HIP: return "QL_E_HIP";
    case QL_E_STATE: return "QL_E_STATE";
    default: return "QL_E_UNKNOWN";
    }
}

/* returns 1 (and throws) when rc is an error */
static inline int throw_rc(napi_env env, int rc)
{
    if (rc == QL_OK) return 0;
    char msg[600];
    snprintf(msg, sizeof msg, "%s: %s", code_name(rc), ql_last_error());
    napi_throw_error(env, code_name(rc), msg);
    return 1;
}

static inline int get_args(napi_env env, napi_callback_info info, size_t want, napi_value* argv)
{
    size_t argc = want;
    if (napi_get_cb_info(env, info, &argc, argv, NULL, NULL) != napi_ok || argc < want) {
        napi_throw_type_error(env, "QL_E_INVALID", "too few arguments");
        return 1;
    }
    return 0;
}

static inline int get_ptr(napi_env env, napi_value v, void** out)
{
    napi_valuetype t;
    if (napi_typeof(env, v, &t) != napi_ok || t != napi_external ||
        napi_get_value_external(env, v, out) != napi_ok) {
        napi_throw_type_error(env, "QL_E_INVALID", "expected a qlinear handle");
        return 1;
    }
    return 0;
}

static inline int get_i32(napi_env env, napi_value v, int32_t* out)
{
    if (napi_get_value_int32(env, v, out) != napi_ok) {
        napi_throw_type_error(env, "QL_E_INVALID", "expected an integer");
        return 1;
    }
    return 0;
}

/* non-negative integer offset/size as a JS number; null/undefined -> QL_NONE when allow_none */
static inline int get_u64(napi_env env, napi_value v, uint64_t* out, int allow_none)
{
    napi_valuetype t;
    napi_typeof(env, v, &t);
    if (allow_none && (t == napi_null || t == napi_undefined)) {
        *out = QL_NONE;
        return 0;
    }
    double d;
    if (t != napi_number || napi_get_value_double(env, v, &d) != napi_ok || d < 0 ||
        d > 9007199254740992.0 || d != (double)(uint64_t)d) {
        napi_throw_type_error(env, "QL_E_INVALID", "expected a non-negative integer");
        return 1;
    }
    *out = (uint64_t)d;
    return 0;
}

static inline napi_value make_u64(napi_env env, uint64_t v)
{
    napi_value r;
    napi_create_double(env, (double)v, &r);
    return r;
}

static inline napi_value make_i32(napi_env env, int32_t v)
{
    napi_value r;
    napi_create_int32(env, v, &r);
    return r;
}

static inline int prop(napi_env env, napi_value obj, const char* name, napi_value* out)
{
    if (napi_get_named_property(env, obj, name, out) != napi_ok) {
        napi_throw_type_error(env, "QL_E_INVALID", name);
        return 1;
    }
    return 0;
}

static inline int get_u64_array(napi_env env, napi_value arr, uint64_t* out, uint32_t n)
{
    uint32_t m;
    if (napi_get_array_length(env, arr, &m) != napi_ok || m != n) {
        napi_throw_type_error(env, "QL_E_INVALID", "offset array length mismatch");
        return 1;
    }
    for (uint32_t i = 0; i < n; i++) {
        napi_value e;
        if (napi_get_element(env, arr, i, &e) != napi_ok || get_u64(env, e, &out[i], 0)) return 1;
    }
    return 0;
}

/* {tableOff, maxPos, nHead, nKvHead, D, rotDim, interleaved, qNormOff|null, kNormOff|null, normEps, qStride, kStride, vStride,
 *  cacheDtype} -> ql_rope_desc */
static inline int get_rope(napi_env env, napi_value obj, ql_rope_desc* d)
{
    const struct {
        const char* name;
        int32_t* out;
    } ints[] = {{"maxPos", &d->max_pos}, {"nHead", &d->n_head}, {"nKvHead", &d->n_kv_head}, {"D", &d->D}, {"rotDim", &d->rot_dim},
                {"interleaved", &d->interleaved}, {"qStride", &d->q_stride}, {"kStride", &d->k_stride}, {"vStride", &d->v_stride},
                {"cacheDtype", &d->cache_dtype}};
    napi_value v;
    double eps;
    memset(d, 0, sizeof *d);
    if (prop(env, obj, "tableOff", &v) || get_u64(env, v, &d->table_off, 0)) return 1;
    if (prop(env, obj, "qNormOff", &v) || get_u64(env, v, &d->q_norm_off, 1)) return 1;
    if (prop(env, obj, "kNormOff", &v) || get_u64(env, v, &d->k_norm_off, 1)) return 1;
    for (size_t i = 0; i < sizeof ints / sizeof ints[0]; i++)
        if (prop(env, obj, ints[i].name, &v) || get_i32(env, v, ints[i].out)) return 1;
    if (prop(env, obj, "normEps", &v) || napi_get_value_double(env, v, &eps) != napi_ok) {
        napi_throw_type_error(env, "QL_E_INVALID", "normEps");
        return 1;
    }
    d->norm_eps = (float)eps;
    return 0;
}
