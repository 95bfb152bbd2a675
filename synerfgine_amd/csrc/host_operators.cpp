// host_operators.cpp -- argument checks of the operators in operators.h, and the calls of their launchers.  Arguments are
// checked before the context is looked at, and nothing is enqueued by a call that is refused.
#include "host_operators.h"

namespace sng_host {

namespace {

void refuse(bool bad, const char* what) {
    if (bad) throw SngError(SNG_ERR_INVALID, what);
}
void check_type(int32_t dtype, bool with_i8) {
    if (dtype < SNG_F16 || dtype > (with_i8 ? SNG_I8 : SNG_F32))
        throw SngError(SNG_ERR_INVALID, with_i8 ? "dtype must be SNG_F16, SNG_BF16, SNG_F32 or SNG_I8" : "dtype must be SNG_F16, SNG_BF16 or SNG_F32");
}
uint64_t elem_bytes(int32_t dtype) { return dtype == SNG_F32 ? 4 : dtype == SNG_I8 ? 1 : 2; }
// pointers hold whole elements of their type
void check_aligned(const void* p, uint64_t bytes, const char* what) { refuse((uint64_t)p % bytes != 0, what); }

void check_choices(uint32_t n, uint32_t k) {
    refuse(k == 0, "k must be at least 1");
    refuse((uint64_t)n * k > CHOICES_MAX, "n * k must be at most 2^28");
}
void check_experts(uint32_t n_experts) {
    refuse(n_experts == 0 || n_experts > EXPERTS_MAX, "n_experts must be 1 to 4096");
}
// rows of d elements with stride ld: the last element's byte offset fits 63 bits
void check_rows(uint32_t d, uint64_t ld, const char* what) {
    refuse(d == 0 || d > (1u << 20), "the row length must be 1 to 2^20");
    refuse(ld < d || ld > (1ull << 31), what);
}

// The device of the context for the call's launches, and the caller's again afterwards
struct OnDevice {
    int before = -1, now;
    explicit OnDevice(sng_ctx* c) : now(c ? c->device : -1) {
        if (!c) throw SngError(SNG_ERR_INVALID, "null context");
        HIPCHK(hipGetDevice(&before));
        if (before != now) HIPCHK(hipSetDevice(now));
    }
    ~OnDevice() {
        if (before >= 0 && before != now) (void)hipSetDevice(before);
    }
};

uint64_t padded(uint64_t n_in) { return (n_in + I8_PAD - 1) / I8_PAD * I8_PAD; }

void check_linear(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts) {
    refuse(n_in == 0 || n_in > I8_IN_MAX, "n_in must be 1 to 131071 (larger sums can overflow 32 bits)");
    refuse(n_out == 0 || n_out > (1u << 20), "n_out must be 1 to 2^20");
    refuse(rows > (1u << 30), "rows must be at most 2^30");
    check_experts(n_experts);
}

// The workspace of a call whose x is brought to 8 bits before the product: the rows, padded; their scales; and where n_in is
// no multiple of 16, the weights in rows that the tiles can take (2 bytes moved a weight, where unaligned tiles took 4 to 10
// times the time of aligned ones); and the sums of the parts of n_in where few tiles share a long one
struct LinearLayout { uint64_t scale, w, partial, bytes; };
LinearLayout linear_i8_layout(uint64_t rows, uint64_t n_in, uint64_t n_out, uint64_t n_experts) {
    LinearLayout l;
    l.scale = rows * padded(n_in);
    l.w = l.scale + (rows * sizeof(float) + 15) / 16 * 16;
    l.partial = l.w;
    if (n_in % 16 != 0 && linear_i8_kernel((uint32_t)rows, (uint32_t)n_in, (uint32_t)n_out, (uint32_t)n_experts) == LinearKernel::Tile) l.partial += n_experts * n_out * padded(n_in);
    l.bytes = l.partial + linear_i8_split((uint32_t)rows, (uint32_t)n_in, (uint32_t)n_out, (uint32_t)n_experts).bytes;
    return l;
}

}  // namespace

uint64_t expert_sort_workspace(uint32_t n, uint32_t k, uint32_t n_experts) {
    check_choices(n, k);
    check_experts(n_experts);
    const uint64_t total = (uint64_t)n * k;
    if (sort_in_one(total, n_experts)) return 0;
    return ((uint64_t)sort_blocks(total) + 1) * n_experts * sizeof(uint32_t);
}

void expert_sort(sng_ctx* c, const int32_t* experts, uint32_t n, uint32_t k, uint32_t n_experts, int32_t* offsets, int32_t* order, int32_t* slot,
                 void* workspace, uint64_t workspace_bytes, hipStream_t s) {
    const uint64_t need = expert_sort_workspace(n, k, n_experts);
    refuse(!offsets || (n && (!experts || !order || !slot)), "null argument");
    for (const void* p : {(const void*)experts, (const void*)offsets, (const void*)order, (const void*)slot, (const void*)workspace})
        check_aligned(p, 4, "the arrays must be aligned to 4 bytes");
    refuse(need > 0 && (!workspace || workspace_bytes < need), "the workspace is smaller than sng_expert_sort_workspace says");
    OnDevice on(c);
    launch_expert_sort(SortArgs{experts, n * k, n_experts, offsets, order, slot, (uint32_t*)workspace}, s);
    HIPCHK(hipGetLastError());
}

void expert_dispatch(sng_ctx* c, const void* x, int32_t dtype, uint32_t d, uint64_t ld_x, const int32_t* order, const int32_t* slot, uint32_t n, uint32_t k, void* rows,
                     uint64_t ld_rows, hipStream_t s) {
    check_choices(n, k);
    check_type(dtype, true);
    check_rows(d, ld_x, "ld_x must be at least d and at most 2^31");
    check_rows(d, ld_rows, "ld_rows must be at least d and at most 2^31");
    refuse(n && (!x || !order || !slot || !rows), "null argument");
    for (const void* p : {x, (const void*)rows}) check_aligned(p, elem_bytes(dtype), "rows must be aligned to their type");
    for (const int32_t* p : {order, slot}) check_aligned(p, 4, "the plan must be aligned to 4 bytes");
    OnDevice on(c);
    if (n == 0) return;
    RowsArgs a{};
    a.src = x; a.ld_src = ld_x; a.dst = rows; a.ld_dst = ld_rows; a.slot = slot; a.n = n; a.k = k; a.d = d; a.dtype = dtype;
    launch_expert_dispatch(a, s);
    HIPCHK(hipGetLastError());
}

void expert_combine(sng_ctx* c, const void* rows, int32_t dtype, uint32_t d, uint64_t ld_rows, const float* weights, const int32_t* slot, uint32_t n, uint32_t k, void* y,
                    uint64_t ld_y, hipStream_t s) {
    check_choices(n, k);
    check_type(dtype, false);
    check_rows(d, ld_rows, "ld_rows must be at least d and at most 2^31");
    check_rows(d, ld_y, "ld_y must be at least d and at most 2^31");
    refuse(n && (!rows || !slot || !y), "null argument");
    for (const void* p : {rows, (const void*)y}) check_aligned(p, elem_bytes(dtype), "rows must be aligned to their type");
    for (const void* p : {(const void*)weights, (const void*)slot}) check_aligned(p, 4, "weights and slot must be aligned to 4 bytes");
    OnDevice on(c);
    if (n == 0) return;
    RowsArgs a{};
    a.src = rows; a.ld_src = ld_rows; a.dst = y; a.ld_dst = ld_y; a.weights = weights; a.slot = slot; a.n = n; a.k = k; a.d = d; a.dtype = dtype;
    launch_expert_combine(a, s);
    HIPCHK(hipGetLastError());
}

void expert_combine_backward(sng_ctx* c, const void* dy, uint64_t ld_dy, const void* rows, uint64_t ld_rows, int32_t dtype, uint32_t d, const float* weights,
                             const int32_t* slot, uint32_t n, uint32_t k, void* drows, uint64_t ld_drows, float* dweights, hipStream_t s) {
    check_choices(n, k);
    check_type(dtype, false);
    check_rows(d, ld_dy, "ld_dy must be at least d and at most 2^31");
    if (dweights) check_rows(d, ld_rows, "ld_rows must be at least d and at most 2^31");
    if (drows) check_rows(d, ld_drows, "ld_drows must be at least d and at most 2^31");
    refuse(!drows && !dweights, "neither gradient is asked for");
    refuse(n && (!dy || !slot || (dweights && !rows)), "null argument");
    for (const void* p : {dy, rows, (const void*)drows}) check_aligned(p, elem_bytes(dtype), "rows must be aligned to their type");
    for (const void* p : {(const void*)weights, (const void*)slot, (const void*)dweights}) check_aligned(p, 4, "weights, slot and dweights must be aligned to 4 bytes");
    OnDevice on(c);
    if (n == 0) return;
    RowsArgs a{};
    a.src = dweights ? rows : nullptr; a.ld_src = dweights ? ld_rows : 0; a.dst = drows; a.ld_dst = drows ? ld_drows : 0; a.dy = dy; a.ld_dy = ld_dy;
    a.weights = weights; a.dweights = dweights; a.slot = slot; a.n = n; a.k = k; a.d = d; a.dtype = dtype;
    launch_expert_combine_backward(a, s);
    HIPCHK(hipGetLastError());
}

void quantize_rows_i8(sng_ctx* c, const void* x, int32_t dtype, uint32_t rows, uint32_t cols, uint64_t ld_x, int8_t* q, uint64_t ld_q, float* scale, hipStream_t s) {
    check_type(dtype, false);
    check_rows(cols, ld_x, "ld_x must be at least cols and at most 2^31");
    check_rows(cols, ld_q, "ld_q must be at least cols and at most 2^31");
    refuse(rows > (1u << 30), "rows must be at most 2^30");
    refuse(rows && (!x || !q || !scale), "null argument");
    check_aligned(x, elem_bytes(dtype), "rows must be aligned to their type");
    check_aligned(scale, 4, "scale must be aligned to 4 bytes");
    OnDevice on(c);
    if (rows == 0) return;
    launch_quantize_rows(QuantArgs{x, ld_x, dtype, rows, cols, cols, q, ld_q, scale}, s);
    HIPCHK(hipGetLastError());
}

uint64_t linear_i8_workspace(uint32_t rows, uint32_t n_in, uint32_t n_out, int32_t x_dtype, uint32_t n_experts) {
    check_linear(rows, n_in, n_out, n_experts);
    check_type(x_dtype, true);
    if (rows == 0 || x_dtype == SNG_I8 || linear_i8_quantizes(rows, n_in, n_out, n_experts)) return 0;
    return linear_i8_layout(rows, n_in, n_out, n_experts).bytes;
}

void linear_i8(sng_ctx* c, const sng_linear_i8_args* p, hipStream_t s) {
    refuse(!p, "null argument");
    const sng_linear_i8_args& a = *p;
    const uint64_t need = linear_i8_workspace(a.rows, a.n_in, a.n_out, a.x_dtype, a.n_experts);
    check_type(a.y_dtype, false);
    refuse(a.ld_x < a.n_in || a.ld_x > (1ull << 31), "ld_x must be at least n_in and at most 2^31");
    refuse(a.ld_w < a.n_in || a.ld_w > (1ull << 31), "ld_w must be at least n_in and at most 2^31");
    refuse(a.ld_y < a.n_out || a.ld_y > (1ull << 31), "ld_y must be at least n_out and at most 2^31");
    refuse(a.relu != 0 && a.relu != 1, "relu must be 0 or 1");
    refuse(!a.d_offsets && a.n_experts != 1, "several experts need their offsets");
    refuse(a.rows && (!a.d_x || !a.d_w || !a.d_w_scale || !a.d_y || (a.x_dtype == SNG_I8 && !a.d_x_scale)), "null argument");
    check_aligned(a.d_x, elem_bytes(a.x_dtype), "x must be aligned to its type");
    check_aligned(a.d_y, elem_bytes(a.y_dtype), "y must be aligned to its type");
    for (const void* q : {(const void*)a.d_x_scale, (const void*)a.d_w_scale, (const void*)a.d_bias, (const void*)a.d_offsets})
        check_aligned(q, 4, "scales, bias and offsets must be aligned to 4 bytes");
    refuse((uint64_t)a.d_workspace % 16 != 0, "the workspace must be aligned to 16 bytes");
    refuse(a.rows && need > 0 && (!a.d_workspace || a.workspace_bytes < need), "the workspace is smaller than sng_linear_i8_workspace says");
    OnDevice on(c);
    if (a.rows == 0) return;
    LinearArgs l{};
    l.x = a.d_x; l.ld_x = a.ld_x; l.x_dtype = a.x_dtype; l.x_scale = a.d_x_scale; l.w = a.d_w; l.ld_w = a.ld_w; l.w_scale = a.d_w_scale; l.bias = a.d_bias;
    l.offsets = a.d_offsets; l.n_experts = a.n_experts; l.rows = a.rows; l.n_in = a.n_in; l.n_out = a.n_out; l.y = a.d_y; l.ld_y = a.ld_y;
    l.y_dtype = a.y_dtype; l.relu = a.relu;
    l.kernel = linear_i8_kernel(a.rows, a.n_in, a.n_out, a.n_experts);
    if (need) {
        const LinearLayout at = linear_i8_layout(a.rows, a.n_in, a.n_out, a.n_experts);
        const uint64_t ld = padded(a.n_in);
        int8_t* q = (int8_t*)a.d_workspace;
        float* scale = (float*)(q + at.scale);
        launch_quantize_rows(QuantArgs{a.d_x, a.ld_x, a.x_dtype, a.rows, a.n_in, (uint32_t)ld, q, ld, scale}, s);
        HIPCHK(hipGetLastError());
        l.splits = linear_i8_split(a.rows, a.n_in, a.n_out, a.n_experts).splits; l.partial = (int32_t*)(q + at.partial);
        l.x = q; l.ld_x = ld; l.x_dtype = SNG_I8; l.x_scale = scale;
        if (at.partial > at.w) {
            launch_pad_rows(a.d_w, a.ld_w, a.n_in, (uint64_t)a.n_experts * a.n_out, (uint32_t)ld, q + at.w, s);
            HIPCHK(hipGetLastError());
            l.w = q + at.w; l.ld_w = ld; l.n_in = (uint32_t)ld;   // (zeros behind the rows on both sides)
        }
    }
    launch_linear_i8(l, s);
    HIPCHK(hipGetLastError());
}

}  // namespace sng_host
