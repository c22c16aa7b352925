// extern "C" entry points of serving in 8 bits (declared in include/tsfm_attn.h): argument checks, then one or
// two launches on the caller's stream. Nothing is allocated, kept or waited for.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/tsfm_attn.h"
#include "abi_internal.hpp"
#include "kv8.hpp"
#include "launch.hpp"

using tsfm::abi::aligned;
using tsfm::abi::ensure_ready;
using tsfm::abi::fail;
using tsfm::abi::hip_fail;

static_assert(tsfm::kKvBlock == TSFM_KV8_BLOCK && tsfm::kCodeE4m3 == TSFM_CODE_E4M3 && tsfm::kCodeI8 == TSFM_CODE_I8,
              "the kernels' constants are the ABI's");

namespace {

constexpr int64_t kMaxSpan = (int64_t)1 << 46;       // elements of any array or strided view
constexpr int32_t kMaxWidth = (1 << 25) - 1;         // blocks of a request: positions stay below 2^31
constexpr int32_t kMaxTokens = 1 << 30;
constexpr int64_t kMaxRowBytes = (int64_t)1 << 23;   // 256 rows of a product's operand stay below 2 GiB

// The product of the factors (all >= 0), or kMaxSpan + 1 where it passes kMaxSpan.
int64_t volume(std::initializer_list<int64_t> factors) {
    int64_t v = 1;
    for (const int64_t f : factors)
        if (__builtin_mul_overflow(v, f, &v) || v > kMaxSpan) v = kMaxSpan + 1;
    return v;
}

// Elements that `rows` rows of `width`, `ld` apart, span; kMaxSpan + 1 where that passes kMaxSpan.
int64_t rows_span(int64_t rows, int64_t ld, int64_t width) {
    const int64_t v = rows > 0 ? volume({rows - 1, ld}) : 0;
    return v > kMaxSpan || width > kMaxSpan - v ? kMaxSpan + 1 : v + width;
}

int check_flags(uint32_t flags) {
    if (flags & ~TSFM_ATTN_DEVICE_PTRS) return fail(TSFM_E_INVALID, "unknown flags %#x", flags);
    if (!(flags & TSFM_ATTN_DEVICE_PTRS)) return fail(TSFM_E_UNSUPPORTED, "8-bit serving takes device pointers only");
    return TSFM_OK;
}

int check_requests(int32_t requests, int32_t blocks, int32_t width) {
    if (requests < 1 || blocks < 1 || width < 1) return fail(TSFM_E_INVALID, "requests, blocks and table_width must be positive");
    if (requests > TSFM_KV8_MAX_REQUESTS)
        return fail(TSFM_E_UNSUPPORTED, "%d requests (supported: %d)", requests, TSFM_KV8_MAX_REQUESTS);
    if (width > kMaxWidth) return fail(TSFM_E_UNSUPPORTED, "table_width %d (supported: %d)", width, kMaxWidth);
    if (blocks > INT32_MAX / 2) return fail(TSFM_E_UNSUPPORTED, "%d blocks (supported: %d)", blocks, INT32_MAX / 2);
    return TSFM_OK;
}

int check_cache(const tsfm_kv8_cache& c, bool pointers) {
    if (c.dtype != TSFM_DTYPE_BF16 && c.dtype != TSFM_DTYPE_F16)
        return fail(TSFM_E_UNSUPPORTED, "the 8-bit cache takes bf16 and f16 tokens");
    if (c.code != TSFM_CODE_E4M3 && c.code != TSFM_CODE_I8) return fail(TSFM_E_INVALID, "bad code %d", c.code);
    if (c.head_dim != 64 && c.head_dim != 128)
        return fail(TSFM_E_UNSUPPORTED, "head_dim %d (supported: 64, 128)", c.head_dim);
    if (c.kv_heads < 1) return fail(TSFM_E_INVALID, "kv_heads must be positive");
    const int rc = check_requests(c.requests, c.blocks, c.table_width);
    if (rc != TSFM_OK) return rc;
    const int64_t row = (int64_t)64 * c.head_dim;
    if (volume({c.blocks, c.kv_heads, row}) > kMaxSpan || volume({c.requests, c.kv_heads, row}) > kMaxSpan)
        return fail(TSFM_E_UNSUPPORTED, "the cache spans more than 2^46 elements");
    if (!pointers) return TSFM_OK;
    if (c.k == nullptr || c.v == nullptr || c.scales == nullptr || c.k_tail == nullptr || c.v_tail == nullptr ||
        c.table == nullptr || c.len == nullptr)
        return fail(TSFM_E_INVALID, "the cache's arrays are required");
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_tail, 16) || !aligned(c.v_tail, 16) ||
        !aligned(c.scales, 8) || !aligned(c.table, 4) || !aligned(c.len, 4))
        return fail(TSFM_E_UNSUPPORTED, "the cache's k, v and tails must be 16-byte, its scales 8-byte aligned");
    return TSFM_OK;
}

tsfm::Kv8 view(const tsfm_kv8_cache& c) {
    tsfm::Kv8 v{};
    v.k = static_cast<uint8_t*>(c.k);
    v.v = static_cast<uint8_t*>(c.v);
    v.scales = c.scales;
    v.k_tail = static_cast<uint16_t*>(c.k_tail);
    v.v_tail = static_cast<uint16_t*>(c.v_tail);
    v.table = c.table;
    v.len = c.len;
    v.requests = c.requests;
    v.heads = c.kv_heads;
    v.blocks = c.blocks;
    v.width = c.table_width;
    return v;
}

// The stream's device, current while the call queues its kernels (a launch on another device's stream fails).
class OnDeviceOf {
public:
    explicit OnDeviceOf(void* stream) {
        hipDevice_t dev = 0;
        // The NULL stream is the current device's; so are hipStreamLegacy and hipStreamPerThread (1 and 2).
        if (reinterpret_cast<uintptr_t>(stream) <= 2 ||
            hipStreamGetDevice(static_cast<hipStream_t>(stream), &dev) != hipSuccess || hipGetDevice(&was_) != hipSuccess ||
            was_ == dev)
            was_ = -1;
        else if (hipSetDevice(dev) != hipSuccess)
            was_ = -1;
    }
    ~OnDeviceOf() {
        if (was_ >= 0) (void)hipSetDevice(was_);
    }
    OnDeviceOf(const OnDeviceOf&) = delete;
    OnDeviceOf& operator=(const OnDeviceOf&) = delete;

private:
    int was_ = -1;
};

// Checks an attend call and fills its parameters, split included; *need: bytes of workspace.
int attend_request(const tsfm_kv8_attend_args* a, tsfm::Kv8Attend* p, int64_t* need, bool pointers) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if ((rc = check_cache(a->cache, pointers)) != TSFM_OK) return rc;
    const int32_t hd = a->cache.head_dim;
    if (a->heads < 1 || a->heads % a->cache.kv_heads)
        return fail(TSFM_E_INVALID, "heads %d is no multiple of kv_heads %d", a->heads, a->cache.kv_heads);
    if (a->max_tokens < 0 || a->max_new < 0 || a->max_len < 0) return fail(TSFM_E_INVALID, "negative size");
    if (a->max_tokens > kMaxTokens) return fail(TSFM_E_UNSUPPORTED, "%d tokens (supported: %d)", a->max_tokens, kMaxTokens);
    if (!(a->scale >= 0.f)) return fail(TSFM_E_UNSUPPORTED, "attention needs a non-negative scale");
    const int64_t row = volume({a->heads, hd});
    if (row > INT32_MAX) return fail(TSFM_E_UNSUPPORTED, "a token's heads span more than 2^31 elements");
    if (pointers) {
        if (a->cu_tokens == nullptr || a->q == nullptr || a->o == nullptr)
            return fail(TSFM_E_INVALID, "cu_tokens, q and o are required");
        if (a->q_tok < 0 || a->o_tok < 0) return fail(TSFM_E_INVALID, "negative stride");
        if (a->o_tok < row && a->max_tokens > 1) return fail(TSFM_E_INVALID, "o token stride smaller than heads * head_dim");
        if (a->q_tok % 8 || a->o_tok % 8) return fail(TSFM_E_UNSUPPORTED, "strides must be multiples of 16 bytes");
        if (rows_span(a->max_tokens, a->q_tok, row) > kMaxSpan || rows_span(a->max_tokens, a->o_tok, row) > kMaxSpan)
            return fail(TSFM_E_UNSUPPORTED, "a q/o view spans more than 2^46 elements");
        if (!aligned(a->q, 16) || !aligned(a->o, 16) || !aligned(a->cu_tokens, 4))
            return fail(TSFM_E_UNSUPPORTED, "q and o must be 16-byte aligned");
    }
    *p = tsfm::Kv8Attend{};
    p->c = view(a->cache);
    p->cu_tokens = a->cu_tokens;
    p->q = static_cast<const uint16_t*>(a->q);
    p->o = static_cast<uint16_t*>(a->o);
    p->q_tok = a->q_tok;
    p->o_tok = a->o_tok;
    p->heads = a->heads;
    p->max_tokens = a->max_tokens;
    p->group = a->heads / a->cache.kv_heads;
    p->c2 = a->scale * tsfm::kLog2e;
    p->part = static_cast<float*>(a->workspace);
    *need = 0;
    if (a->max_tokens == 0) return TSFM_OK;
    const int cus = tsfm::device_cus();
    *need = tsfm::kv8_attend_plan(*p, hd, a->max_new, a->max_len, cus > 0 ? cus : 256);
    if (*need < 0) return fail(TSFM_E_UNSUPPORTED, "too many rows, heads and requests for one launch");
    return TSFM_OK;
}

}  // namespace

extern "C" {

int tsfm_kv8_plan(const tsfm_kv8_plan_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if ((rc = check_requests(a->requests, a->blocks, a->table_width)) != TSFM_OK) return rc;
    if (a->max_tokens < 1 || a->max_items < 1) return fail(TSFM_E_INVALID, "max_tokens and max_items must be positive");
    if (a->max_tokens > kMaxTokens) return fail(TSFM_E_UNSUPPORTED, "%d tokens (supported: %d)", a->max_tokens, kMaxTokens);
    const int32_t items = std::min(a->max_tokens, a->max_tokens / TSFM_KV8_BLOCK + 2 * a->requests);
    if (a->max_items < items) return fail(TSFM_E_INVALID, "max_items %d: this step can touch %d blocks", a->max_items, items);
    if (a->max_items > kMaxTokens) return fail(TSFM_E_UNSUPPORTED, "%d items (supported: %d)", a->max_items, kMaxTokens);
    const void* need[] = {a->n_new, a->len, a->len_out, a->free_list, a->free_count, a->free_count_out, a->table,
                          a->cu_tokens, a->cu_blocks, a->cu_items, a->slots, a->pos, a->items, a->status};
    for (const void* q : need) {
        if (q == nullptr) return fail(TSFM_E_INVALID, "the plan's arrays are required");
        if (!aligned(q, 4)) return fail(TSFM_E_UNSUPPORTED, "the plan's arrays must be aligned to their elements");
    }
    if (!aligned(a->slots, 8) || !aligned(a->items, 8)) return fail(TSFM_E_UNSUPPORTED, "slots and items must be 8-byte aligned");
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    tsfm::Kv8Plan p{};
    p.n_new = a->n_new;
    p.len = a->len;
    p.free_list = a->free_list;
    p.free_count = a->free_count;
    p.len_out = a->len_out;
    p.free_count_out = a->free_count_out;
    p.table = a->table;
    p.cu_tokens = a->cu_tokens;
    p.cu_blocks = a->cu_blocks;
    p.cu_items = a->cu_items;
    p.pos = a->pos;
    p.items = a->items;
    p.status = a->status;
    p.slots = a->slots;
    p.requests = a->requests;
    p.blocks = a->blocks;
    p.width = a->table_width;
    p.max_tokens = a->max_tokens;
    p.max_items = a->max_items;
    OnDeviceOf on(a->stream);
    const hipError_t e = tsfm::launch_kv8_plan(p, static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "plan launch");
}

int tsfm_kv8_release(const tsfm_kv8_release_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if ((rc = check_requests(a->requests, a->blocks, a->table_width)) != TSFM_OK) return rc;
    const void* need[] = {a->len, a->table, a->free_list, a->free_count, a->status};
    if (a->drop == nullptr) return fail(TSFM_E_INVALID, "the release's arrays are required");
    for (const void* q : need) {
        if (q == nullptr) return fail(TSFM_E_INVALID, "the release's arrays are required");
        if (!aligned(q, 4)) return fail(TSFM_E_UNSUPPORTED, "the release's arrays must be aligned to their elements");
    }
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    tsfm::Kv8Release p{};
    p.drop = a->drop;
    p.len = a->len;
    p.table = a->table;
    p.free_list = a->free_list;
    p.free_count = a->free_count;
    p.status = a->status;
    p.requests = a->requests;
    p.blocks = a->blocks;
    p.width = a->table_width;
    OnDeviceOf on(a->stream);
    const hipError_t e = tsfm::launch_kv8_release(p, static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "release launch");
}

int tsfm_kv8_append(const tsfm_kv8_append_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if ((rc = check_cache(a->cache, true)) != TSFM_OK) return rc;
    if (a->max_tokens < 0 || a->max_items < 0) return fail(TSFM_E_INVALID, "negative size");
    if (a->max_tokens > kMaxTokens || a->max_items > kMaxTokens)
        return fail(TSFM_E_UNSUPPORTED, "more than %d tokens or items", kMaxTokens);
    if (a->max_tokens == 0 || a->max_items == 0) return TSFM_OK;
    if (a->cu_tokens == nullptr || a->items == nullptr || a->k == nullptr || a->v == nullptr)
        return fail(TSFM_E_INVALID, "cu_tokens, items, k and v are required");
    if (a->k_tok < 0 || a->v_tok < 0) return fail(TSFM_E_INVALID, "negative stride");
    if (a->k_tok % 8 || a->v_tok % 8) return fail(TSFM_E_UNSUPPORTED, "strides must be multiples of 16 bytes");
    if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cu_tokens, 4) || !aligned(a->items, 4))
        return fail(TSFM_E_UNSUPPORTED, "k and v must be 16-byte aligned");
    const int64_t row = volume({a->cache.kv_heads, a->cache.head_dim});
    if (row > INT32_MAX) return fail(TSFM_E_UNSUPPORTED, "a token's heads span more than 2^31 elements");
    if (rows_span(a->max_tokens, a->k_tok, row) > kMaxSpan || rows_span(a->max_tokens, a->v_tok, row) > kMaxSpan)
        return fail(TSFM_E_UNSUPPORTED, "a k/v view spans more than 2^46 elements");
    if (volume({a->max_items, a->cache.kv_heads}) > INT32_MAX)
        return fail(TSFM_E_UNSUPPORTED, "too many items and heads for one launch");
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    tsfm::Kv8Append p{};
    p.c = view(a->cache);
    p.cu_tokens = a->cu_tokens;
    p.items = a->items;
    p.k = static_cast<const uint16_t*>(a->k);
    p.v = static_cast<const uint16_t*>(a->v);
    p.k_tok = a->k_tok;
    p.v_tok = a->v_tok;
    p.max_tokens = a->max_tokens;
    p.max_items = a->max_items;
    OnDeviceOf on(a->stream);
    const hipError_t e = tsfm::launch_kv8_append(p, a->cache.code, a->cache.dtype == TSFM_DTYPE_BF16, a->cache.head_dim,
                                                 static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "cache append launch");
}

int64_t tsfm_kv8_attend_workspace(const tsfm_kv8_attend_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL"), -1;
    OnDeviceOf on(a->stream);
    tsfm::Kv8Attend p;
    int64_t need = 0;
    return attend_request(a, &p, &need, false) == TSFM_OK ? need : -1;
}

int tsfm_kv8_attend(const tsfm_kv8_attend_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    OnDeviceOf on(a->stream);
    tsfm::Kv8Attend p;
    int64_t need = 0;
    int rc = attend_request(a, &p, &need, true);
    if (rc != TSFM_OK || a->max_tokens == 0) return rc;
    if (need > 0) {
        if (a->workspace == nullptr || a->workspace_bytes < need)
            return fail(TSFM_E_INVALID, "this call needs a workspace of %lld bytes", (long long)need);
        if (!aligned(a->workspace, 16)) return fail(TSFM_E_UNSUPPORTED, "the workspace must be 16-byte aligned");
    }
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    const hipError_t e = tsfm::launch_kv8_attend(p, a->cache.code, a->cache.dtype == TSFM_DTYPE_BF16, a->cache.head_dim,
                                                 static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "cache attention launch");
}

int tsfm_f8_quantize(const tsfm_f8_quantize_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if (a->dtype < TSFM_DTYPE_F32 || a->dtype > TSFM_DTYPE_F16) return fail(TSFM_E_INVALID, "bad dtype %d", a->dtype);
    if (a->group_rows != 1 && a->group_rows != 128)
        return fail(TSFM_E_UNSUPPORTED, "group_rows %d (supported: 1, 128)", a->group_rows);
    if (a->rows < 0 || a->cols < 0 || a->x_ld < 0 || a->codes_ld < 0 || a->scales_ld < 0)
        return fail(TSFM_E_INVALID, "negative size");
    if (a->rows == 0 || a->cols == 0) return TSFM_OK;
    if (a->x == nullptr || a->codes == nullptr || a->scales == nullptr)
        return fail(TSFM_E_INVALID, "x, codes and scales are required");
    if (a->cols % 16) return fail(TSFM_E_UNSUPPORTED, "cols %d is no multiple of 16", a->cols);
    const int64_t groups = ((int64_t)a->cols + 127) / 128, scale_rows = ((int64_t)a->rows + a->group_rows - 1) / a->group_rows;
    if ((a->rows > 1 && a->codes_ld < a->cols) || (scale_rows > 1 && a->scales_ld < groups))
        return fail(TSFM_E_INVALID, "rows of codes or scales overlap");
    if (a->x_ld % (a->dtype == TSFM_DTYPE_F32 ? 4 : 8) || a->codes_ld % 16)
        return fail(TSFM_E_UNSUPPORTED, "row strides of x and codes must be multiples of 16 bytes");
    if (!aligned(a->x, 16) || !aligned(a->codes, 16) || !aligned(a->scales, 4))
        return fail(TSFM_E_UNSUPPORTED, "x and codes must be 16-byte aligned");
    if (rows_span(a->rows, a->x_ld, a->cols) > kMaxSpan || rows_span(a->rows, a->codes_ld, a->cols) > kMaxSpan ||
        rows_span(scale_rows, a->scales_ld, groups) > kMaxSpan)
        return fail(TSFM_E_UNSUPPORTED, "an array spans more than 2^46 elements");
    if (volume({a->rows, groups}) > INT32_MAX) return fail(TSFM_E_UNSUPPORTED, "too many groups for one launch");
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    tsfm::F8Quantize p{};
    p.x = a->x;
    p.codes = a->codes;
    p.scales = a->scales;
    p.x_ld = a->x_ld;
    p.codes_ld = a->codes_ld;
    p.scales_ld = a->scales_ld;
    p.rows = a->rows;
    p.cols = a->cols;
    p.group_rows = a->group_rows;
    OnDeviceOf on(a->stream);
    const hipError_t e = tsfm::launch_f8_quantize(p, a->dtype, static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "quantisation launch");
}

int tsfm_f8_gemm_nt(const tsfm_f8_gemm_args* a) {
    if (a == nullptr) return fail(TSFM_E_INVALID, "args is NULL");
    int rc = check_flags(a->flags);
    if (rc != TSFM_OK) return rc;
    if (a->out_dtype < TSFM_DTYPE_F32 || a->out_dtype > TSFM_DTYPE_F16)
        return fail(TSFM_E_INVALID, "bad out_dtype %d", a->out_dtype);
    if (a->m < 0 || a->n < 0 || a->k < 0 || a->a_ld < 0 || a->b_ld < 0 || a->a_scales_ld < 0 || a->b_scales_ld < 0 || a->c_ld < 0)
        return fail(TSFM_E_INVALID, "negative size");
    if (a->m == 0 || a->n == 0) return TSFM_OK;
    if (a->k == 0) return fail(TSFM_E_UNSUPPORTED, "k must be positive");
    if (a->a == nullptr || a->b == nullptr || a->a_scales == nullptr || a->b_scales == nullptr || a->c == nullptr)
        return fail(TSFM_E_INVALID, "a, b, their scales and c are required");
    if (a->k % 16) return fail(TSFM_E_UNSUPPORTED, "k %d is no multiple of 16", a->k);
    if (a->m > 1 && a->c_ld < a->n) return fail(TSFM_E_INVALID, "rows of c overlap");
    if (a->a_ld % 16 || a->b_ld % 16) return fail(TSFM_E_UNSUPPORTED, "row strides of a and b must be multiples of 16 bytes");
    if (std::max({a->a_ld, a->b_ld, (int64_t)a->k}) > kMaxRowBytes)
        return fail(TSFM_E_UNSUPPORTED, "rows of a and b are at most 2^23 bytes");
    if (!aligned(a->a, 16) || !aligned(a->b, 16) || !aligned(a->a_scales, 4) || !aligned(a->b_scales, 4) ||
        !aligned(a->c, a->out_dtype == TSFM_DTYPE_F32 ? 4 : 2))
        return fail(TSFM_E_UNSUPPORTED, "a and b must be 16-byte aligned, scales and c to their elements");
    const int64_t kb = ((int64_t)a->k + 127) / 128;
    if (rows_span(a->m, a->a_ld, a->k) > kMaxSpan || rows_span(a->n, a->b_ld, a->k) > kMaxSpan ||
        rows_span(a->m, a->a_scales_ld, kb) > kMaxSpan || rows_span(((int64_t)a->n + 127) / 128, a->b_scales_ld, kb) > kMaxSpan ||
        rows_span(a->m, a->c_ld, a->n) > kMaxSpan)
        return fail(TSFM_E_UNSUPPORTED, "an array spans more than 2^46 elements");
    if ((rc = ensure_ready()) != TSFM_OK) return rc;
    tsfm::F8Gemm p{};
    p.a = a->a;
    p.b = a->b;
    p.a_scales = a->a_scales;
    p.b_scales = a->b_scales;
    p.c = a->c;
    p.a_ld = a->a_ld;
    p.b_ld = a->b_ld;
    p.a_scales_ld = a->a_scales_ld;
    p.b_scales_ld = a->b_scales_ld;
    p.c_ld = a->c_ld;
    p.m = a->m;
    p.n = a->n;
    p.k = a->k;
    OnDeviceOf on(a->stream);
    const int cus = tsfm::device_cus();
    const hipError_t e = tsfm::launch_f8_gemm(p, a->out_dtype, cus > 0 ? cus : 256, static_cast<hipStream_t>(a->stream));
    return e == hipSuccess ? TSFM_OK : hip_fail(e, "8-bit product launch");
}

}  // extern "C"
