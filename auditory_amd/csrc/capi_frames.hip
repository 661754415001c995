// C ABI of the feature-map and frame-sequence operators: argument checks, routes and launches (group_norm.hip,
// causal_conv.hip, scan.hip, scan_grad.hip).  Nothing here allocates, synchronises or keeps a pointer.
#include "capi_internal.h"
#include "frame_ops.h"

using namespace audc;

namespace {

constexpr int64_t kMaxElements = int64_t(1) << 40;
constexpr int32_t kMaxRows = 1 << 30;  // rows of an item: a tile behind them still counts in 32 bits
constexpr int32_t kMaxChannels = 1 << 24;
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

// the context's device for the length of a call; the caller's current device is put back
struct OnDevice {
    int before = -1;
    bool changed = false;
    hipError_t err = hipSuccess;
    explicit OnDevice(const aud_ctx* c) {
        if (hipGetDevice(&before) == hipSuccess && before == c->device) return;
        err = hipSetDevice(c->device);
        changed = err == hipSuccess && before >= 0;
    }
    ~OnDevice() {
        if (changed) (void)hipSetDevice(before);
    }
};

int elem_bytes(int dtype) { return dtype == AUD_F32 ? 4 : 2; }
bool known_type(int dtype) { return dtype == AUD_F32 || dtype == AUD_BF16 || dtype == AUD_F16; }

// an input [items, rows, width] with its strides: no two elements in one place, items or rows outermost
struct Input {
    const void* p;
    int64_t items, rows, width, item, row;
    bool strides_ok() const {
        if (items == 0 || rows == 0) return true;
        if (rows > 1 && (row < width || row > kMaxElements / (rows - 1))) return false;
        if (items > 1 && (item < width || item > kMaxElements / (items - 1))) return false;
        return items <= 1 || rows <= 1 || item >= (rows - 1) * row + width || row >= (items - 1) * item + width;
    }
    // bytes from p to the end of the last element
    int64_t span(int e) const { return items && rows && width ? ((items - 1) * item + (rows - 1) * row + width) * e : 0; }
    bool aligned(int bytes, int e) const {
        if (!p) return true;
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows <= 1 || row * e % bytes == 0) && (items <= 1 || item * e % bytes == 0);
    }
};
template <typename F>
int alignment(int e, F&& fits) {  // the largest of 16, 8, 4 (and e) bytes that fits() says everything is a multiple of
    for (int b = 16; b > e; b /= 2)
        if (fits(b)) return b;
    return e;
}
bool at(const void* p, int bytes) { return !p || reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && na > 0 && nb > 0 && x < y + uintptr_t(nb) && y < x + uintptr_t(na);
}

struct Range {
    const void* p;
    int64_t bytes;
};
// an output on an input, or on another output
bool clash(const Range* outs, int n_out, const Range* ins, int n_in) {
    for (int i = 0; i < n_out; ++i) {
        for (int j = 0; j < n_in; ++j)
            if (overlap(outs[i].p, outs[i].bytes, ins[j].p, ins[j].bytes)) return true;
        for (int j = i + 1; j < n_out; ++j)
            if (overlap(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return true;
    }
    return false;
}

int workspace_ok(aud_ctx* c, const void* ws, int64_t have, int64_t need) {
    if (need == 0) return AUD_OK;
    if (!ws || have < need) return fail(c, AUD_EINVAL, "workspace too small");
    if (!at(ws, 16)) return fail(c, AUD_EINVAL, "workspace must be 16-byte aligned");
    return AUD_OK;
}

// ---- group norm ----
const char* norm_bad(const aud_norm_params* p, bool grad) {
    if (!p) return "null parameters";
    if (!known_type(p->dtype)) return "dtype must be AUD_F32, AUD_BF16 or AUD_F16";
    if (p->act < AUD_ACT_NONE || p->act > AUD_ACT_GELU) return "unknown activation";
    if (p->n_items < 0 || p->rows < 0 || p->rows > kMaxRows || p->channels < 1 || p->groups < 1) return "bad shape";
    if (p->channels > 4096) return "group norm takes at most 4096 channels";
    if (p->channels % p->groups) return "channels must be a multiple of groups";
    if (!(p->eps > 0.f)) return "eps must be positive";
    if (int64_t(p->n_items) * p->rows > kMaxElements / p->channels) return "tensor too large";
    const Input x{nullptr, p->n_items, p->rows, p->channels, p->x_item, p->x_row};
    const Input d{nullptr, p->n_items, p->rows, p->channels, p->dy_item, p->dy_row};
    if (!x.strides_ok() || (grad && !d.strides_ok())) return "strides make rows or items overlap, or reach too far";
    return nullptr;
}
// (the route goes by sizes alone, so that the workspace has one size whatever the alignment)
aud::NormRoute norm_route_of(const aud_norm_params* p, int align, bool grad) {
    return aud::norm_route(p->dtype, p->n_items > 0 ? p->n_items : 1, p->rows, p->channels, p->groups, align, grad);
}

// ---- causal convolution ----
const char* conv_bad(const aud_conv_params* p, bool grad) {
    if (!p) return "null parameters";
    if (!known_type(p->dtype)) return "dtype must be AUD_F32, AUD_BF16 or AUD_F16";
    if (p->act != AUD_ACT_NONE && p->act != AUD_ACT_SILU) return "the convolution's activation is AUD_ACT_NONE or AUD_ACT_SILU";
    if (p->n_items < 0 || p->steps < 0 || p->steps > kMaxRows || p->channels < 1 || p->channels > kMaxChannels) return "bad shape";
    if (p->taps < 1 || p->taps > 4) return "taps must be 1 to 4";
    if (int64_t(p->n_items) * p->steps > kMaxElements / p->channels) return "tensor too large";
    const Input x{nullptr, p->n_items, p->steps, p->channels, p->x_item, p->x_row};
    const Input d{nullptr, p->n_items, p->steps, p->channels, p->dy_item, p->dy_row};
    if (!x.strides_ok() || (grad && !d.strides_ok())) return "strides make rows or items overlap, or reach too far";
    return nullptr;
}
int64_t conv_tiles(const aud_conv_params* p, int T) { return p->steps > 0 ? (int64_t(p->steps) + T - 1) / T : 1; }

// ---- selective scan ----
const char* scan_bad(const aud_scan_params* p, bool gated, bool grad) {
    if (!p) return "null parameters";
    if (!known_type(p->dtype)) return "dtype must be AUD_F32, AUD_BF16 or AUD_F16";
    if (p->n_items < 0 || p->steps < 0 || p->steps > kMaxRows || p->channels < 1 || p->channels > kMaxChannels || p->groups < 1) return "bad shape";
    if (p->channels % p->groups) return "channels must be a multiple of groups";
    if (p->states < 1 || p->states > 64) return "states must be 1 to 64";
    if (int64_t(p->n_items) * (p->steps > 0 ? p->steps : 1) > kMaxElements / (int64_t(p->channels) * p->states)) return "tensor too large";
    const int64_t n = p->n_items, l = p->steps, gn = int64_t(p->groups) * p->states;
    const Input in[] = {{nullptr, n, l, p->channels, p->u_item, p->u_row}, {nullptr, n, l, p->channels, p->delta_item, p->delta_row},
                        {nullptr, n, l, gn, p->b_item, p->b_row}, {nullptr, n, l, gn, p->c_item, p->c_row}};
    for (const Input& i : in)
        if (!i.strides_ok()) return "strides make rows or items overlap, or reach too far";
    const Input z{nullptr, n, l, p->channels, p->z_item, p->z_row}, d{nullptr, n, l, p->channels, p->dy_item, p->dy_row};
    if ((gated && !z.strides_ok()) || (grad && !d.strides_ok())) return "strides make rows or items overlap, or reach too far";
    return nullptr;
}
aud::ScanRoute scan_route_of(const aud_scan_params* p, bool grad) {
    return aud::scan_route(p->n_items > 0 ? p->n_items : 1, p->steps, p->channels, p->groups, p->states, grad);
}
int64_t scan_tiles(const aud_scan_params* p) { return (int64_t(p->steps) + aud::kScanTile - 1) / aud::kScanTile; }
int64_t up4(int64_t n) { return (n + 3) & ~int64_t(3); }
struct ScanSpace {  // floats of the workspace: B and C as a table | chunk sums | gradients: dB and dC by block, parameter sums by chunk
    int64_t table, sums, bc, part;
    int64_t all() const { return table + sums + bc + part; }
};
ScanSpace scan_space(const aud_scan_params* p, const aud::ScanRoute& r, bool grad) {
    const int64_t rows = int64_t(p->n_items) * p->groups;
    ScanSpace s{rows * scan_tiles(p) * aud::kScanTile * 2 * aud::scan_padded_states(p->states),
                up4(aud::scan_sums_floats(r, p->n_items, p->channels, p->states)), 0, 0};
    if (grad) {
        s.bc = r.blocks > 1 ? up4(2 * int64_t(r.blocks) * rows * p->steps * p->states) : 0;
        s.part = int64_t(p->n_items) * r.chunks * (p->states + 2) * p->channels;
    } else if (p->steps == 1) {
        s.table = 0;  // (the one-frame kernel)
    }
    return s;
}
void fill_scan(const aud_scan_params* p, const aud::ScanRoute& r, aud::ScanArgs* a) {
    a->B = p->n_items;
    a->L = p->steps;
    a->Dn = p->channels;
    a->G = p->groups;
    a->N = p->states;
    a->softplus = p->softplus;
    a->ui = p->u_item, a->ur = p->u_row, a->ei = p->delta_item, a->er = p->delta_row, a->zi = p->z_item, a->zr = p->z_row;
    a->bi = p->b_item, a->br = p->b_row, a->ci = p->c_item, a->cr = p->c_row, a->yi = p->dy_item, a->yr = p->dy_row;
    a->chunks = r.chunks;
    a->chunk_tiles = r.chunk_tiles;
    a->fold = r.fold;
}

}  // namespace

extern "C" {

int aud_group_norm_workspace_bytes(const aud_norm_params* p, int gradients, int64_t* bytes) {
    if (!bytes || norm_bad(p, gradients != 0)) return AUD_EINVAL;
    const aud::NormRoute r = norm_route_of(p, 16, gradients != 0);
    *bytes = 4 * aud::norm_workspace_floats(r, p->n_items, p->channels, p->groups, gradients != 0);
    return AUD_OK;
}

int aud_group_norm_batch_dev(aud_ctx* c, const aud_norm_params* p, const void* x, const float* weight, const float* bias,
                             const int32_t* lengths, void* y, float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = norm_bad(p, false)) return fail(c, AUD_EINVAL, why);
    if (p->n_items == 0) return AUD_OK;
    const int e = elem_bytes(p->dtype);
    const int64_t n = int64_t(p->n_items) * p->rows * p->channels;
    if (n && (!x || !y)) return fail(c, AUD_EINVAL, "null buffer");
    const Input in{x, p->n_items, p->rows, p->channels, p->x_item, p->x_row};
    if (!in.aligned(e, e) || !at(y, e) || !at(weight, 4) || !at(bias, 4) || !at(stats, 4) || !at(lengths, 4))
        return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    int64_t need = 0;
    (void)aud_group_norm_workspace_bytes(p, 0, &need);
    if (int rc = workspace_ok(c, workspace, workspace_bytes, need)) return rc;
    const int64_t ch = 4 * int64_t(p->channels), st = 8 * int64_t(p->n_items) * p->groups;
    const Range outs[] = {{y, n * e}, {stats, st}, {workspace, need}};
    const Range ins[] = {{x, in.span(e)}, {weight, ch}, {bias, ch}, {lengths, 4 * int64_t(p->n_items)}};
    if (clash(outs, 3, ins, 4)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    const int align = alignment(e, [&](int b) { return in.aligned(b, e) && at(y, b); });
    const aud::NormRoute r = norm_route_of(p, align, false);
    if (int64_t(p->n_items) * r.chunks > kMaxGrid - 64 || int64_t(p->n_items) * (p->channels / 32 + 1) > kMaxGrid) return fail(c, AUD_EINVAL, "too many items");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    aud::NormArgs a{};
    a.x = x, a.weight = weight, a.bias = bias, a.lengths = lengths, a.out = y;
    a.part = static_cast<float*>(workspace);
    a.stats = stats || !r.join ? stats : a.part + (need / 4 - 2 * int64_t(p->n_items) * p->groups);
    a.B = p->n_items, a.S = p->rows, a.C = p->channels, a.G = p->groups;
    a.xi = p->x_item, a.xr = p->x_row, a.eps = p->eps;
    a.chunks = r.chunks, a.chunk_rows = r.chunk_rows;
    AUD_HIP(c, aud::launch_norm(a, r, p->dtype, p->act, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

int aud_group_norm_grad_dev(aud_ctx* c, const aud_norm_params* p, const void* dy, const void* x, const float* stats,
                            const float* weight, const float* bias, const int32_t* lengths, void* dx, float* dweight,
                            float* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = norm_bad(p, true)) return fail(c, AUD_EINVAL, why);
    const int e = elem_bytes(p->dtype);
    const int64_t n = int64_t(p->n_items) * p->rows * p->channels;
    if (n && (!x || !dy || !dx || !stats)) return fail(c, AUD_EINVAL, "null buffer");
    const Input in{x, p->n_items, p->rows, p->channels, p->x_item, p->x_row}, g{dy, p->n_items, p->rows, p->channels, p->dy_item, p->dy_row};
    if (!in.aligned(e, e) || !g.aligned(e, e) || !at(dx, e) || !at(weight, 4) || !at(bias, 4) || !at(stats, 4) || !at(lengths, 4) ||
        !at(dweight, 4) || !at(dbias, 4))
        return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    int64_t need = 0;
    (void)aud_group_norm_workspace_bytes(p, 1, &need);
    if (int rc = workspace_ok(c, workspace, workspace_bytes, need)) return rc;
    const int64_t ch = 4 * int64_t(p->channels);
    const Range outs[] = {{dx, n * e}, {dweight, ch}, {dbias, ch}, {workspace, need}};
    const Range ins[] = {{x, in.span(e)}, {dy, g.span(e)}, {weight, ch}, {bias, ch}, {stats, 8 * int64_t(p->n_items) * p->groups},
                         {lengths, 4 * int64_t(p->n_items)}};
    if (clash(outs, 4, ins, 6)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    if (n == 0) {  // sums over nothing
        if (dweight || dbias)
            AUD_HIP(c, aud::launch_column_sums(nullptr, 0, p->channels, 0, 2, nullptr, dweight, dbias, static_cast<hipStream_t>(stream)));
        return AUD_OK;
    }
    const int align = alignment(e, [&](int b) { return in.aligned(b, e) && g.aligned(b, e) && at(dx, b); });
    const aud::NormRoute r = norm_route_of(p, align, true);
    if (int64_t(p->n_items) * r.chunks > kMaxGrid - 64 || int64_t(p->n_items) * (p->channels / 32 + 1) > kMaxGrid) return fail(c, AUD_EINVAL, "too many items");
    aud::NormArgs a{};
    a.x = x, a.dy = dy, a.weight = weight, a.bias = bias, a.lengths = lengths, a.out = dx;
    a.stats = const_cast<float*>(stats);  // (only read)
    a.part = static_cast<float*>(workspace);
    a.dweight = dweight, a.dbias = dbias;
    a.B = p->n_items, a.S = p->rows, a.C = p->channels, a.G = p->groups;
    a.xi = p->x_item, a.xr = p->x_row, a.di = p->dy_item, a.dr = p->dy_row, a.eps = p->eps;
    a.chunks = r.chunks, a.chunk_rows = r.chunk_rows;
    AUD_HIP(c, aud::launch_norm_grad(a, r, p->dtype, p->act, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

int aud_causal_conv_batch_dev(aud_ctx* c, const aud_conv_params* p, const void* x, const float* weight, const float* bias,
                              const void* state, const int32_t* lengths, void* y, void* state_out, void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = conv_bad(p, false)) return fail(c, AUD_EINVAL, why);
    if (p->n_items == 0) return AUD_OK;
    const int e = elem_bytes(p->dtype);
    const int64_t n = int64_t(p->n_items) * p->steps * p->channels, ns = int64_t(p->n_items) * (p->taps - 1) * p->channels;
    if ((n && (!x || !y)) || !weight) return fail(c, AUD_EINVAL, "null buffer");
    const Input in{x, p->n_items, p->steps, p->channels, p->x_item, p->x_row};
    if (!in.aligned(e, e) || !at(y, e) || !at(state, e) || !at(state_out, e) || !at(weight, 4) || !at(bias, 4) || !at(lengths, 4))
        return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    const int64_t ch = 4 * int64_t(p->channels);
    const Range outs[] = {{y, n * e}, {state_out, ns * e}};
    const Range ins[] = {{x, in.span(e)}, {weight, ch * p->taps}, {bias, ch}, {lengths, 4 * int64_t(p->n_items)},
                         {state == state_out ? nullptr : state, ns * e}};
    if (clash(outs, 2, ins, 5)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    const int align = alignment(e, [&](int b) { return in.aligned(b, e) && at(y, b) && at(state, b) && at(state_out, b); });
    aud::ConvArgs a{};
    a.T = aud::conv_tile(p->dtype, p->n_items, p->steps, p->channels, align);
    if (int64_t(p->n_items) * conv_tiles(p, a.T) > kMaxGrid * 64 / p->channels) return fail(c, AUD_EINVAL, "tensor too large for one call");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    a.x = x, a.weight = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.out = y, a.state_out = state_out;
    a.B = p->n_items, a.L = p->steps, a.D = p->channels, a.xi = p->x_item, a.xr = p->x_row;
    AUD_HIP(c, aud::launch_conv(a, p->dtype, p->act, p->taps, align, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

int aud_causal_conv_workspace_bytes(const aud_conv_params* p, int64_t* bytes) {
    if (!bytes || conv_bad(p, true)) return AUD_EINVAL;
    // the largest of the routes' (by alignment)
    int64_t tiles = 0;
    for (int align = 2; align <= 16; align *= 2)
        tiles = std::max(tiles, conv_tiles(p, aud::conv_tile(p->dtype, p->n_items, p->steps, p->channels, align)));
    *bytes = 4 * int64_t(p->n_items) * tiles * (p->taps + 1) * p->channels;
    return AUD_OK;
}

int aud_causal_conv_grad_dev(aud_ctx* c, const aud_conv_params* p, const void* dy, const void* x, const float* weight,
                             const float* bias, const void* state, const int32_t* lengths, const void* dstate_out, void* dx,
                             float* dweight, float* dbias, void* dstate, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = conv_bad(p, true)) return fail(c, AUD_EINVAL, why);
    const int e = elem_bytes(p->dtype);
    const int64_t n = int64_t(p->n_items) * p->steps * p->channels, ns = int64_t(p->n_items) * (p->taps - 1) * p->channels;
    if ((n && (!x || !dy || !dx)) || !weight) return fail(c, AUD_EINVAL, "null buffer");
    const Input in{x, p->n_items, p->steps, p->channels, p->x_item, p->x_row}, g{dy, p->n_items, p->steps, p->channels, p->dy_item, p->dy_row};
    if (!in.aligned(e, e) || !g.aligned(e, e) || !at(dx, e) || !at(state, e) || !at(dstate_out, e) || !at(dstate, e) || !at(weight, 4) ||
        !at(bias, 4) || !at(lengths, 4) || !at(dweight, 4) || !at(dbias, 4))
        return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    int64_t need = 0;
    (void)aud_causal_conv_workspace_bytes(p, &need);
    if (int rc = workspace_ok(c, workspace, workspace_bytes, need)) return rc;
    const int64_t ch = 4 * int64_t(p->channels);
    const Range outs[] = {{dx, n * e}, {dstate, ns * e}, {dweight, ch * p->taps}, {dbias, ch}, {workspace, need}};
    const Range ins[] = {{x, in.span(e)}, {dy, g.span(e)}, {weight, ch * p->taps}, {bias, ch}, {state, ns * e}, {dstate_out, ns * e},
                         {lengths, 4 * int64_t(p->n_items)}};
    if (clash(outs, 5, ins, 7)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    if (p->n_items == 0) {  // sums over nothing
        if (dweight || dbias)
            AUD_HIP(c, aud::launch_column_sums(nullptr, 0, p->channels, p->taps, 1, dweight, dbias, nullptr, static_cast<hipStream_t>(stream)));
        return AUD_OK;
    }
    const int align = alignment(
        e, [&](int b) { return in.aligned(b, e) && g.aligned(b, e) && at(dx, b) && at(state, b) && at(dstate_out, b) && at(dstate, b); });
    aud::ConvArgs a{};
    a.T = aud::conv_tile(p->dtype, p->n_items, p->steps, p->channels, align);
    if (int64_t(p->n_items) * conv_tiles(p, a.T) > kMaxGrid * 64 / p->channels) return fail(c, AUD_EINVAL, "tensor too large for one call");
    a.x = x, a.dy = dy, a.weight = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.out = dx;
    a.dstate_out = dstate_out, a.dstate = dstate, a.dweight = dweight, a.dbias = dbias, a.part = static_cast<float*>(workspace);
    a.B = p->n_items, a.L = p->steps, a.D = p->channels;
    a.xi = p->x_item, a.xr = p->x_row, a.di = p->dy_item, a.dr = p->dy_row;
    AUD_HIP(c, aud::launch_conv_grad(a, p->dtype, p->act, p->taps, align, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

int aud_scan_workspace_bytes(const aud_scan_params* p, int gradients, int64_t* bytes) {
    if (!bytes || scan_bad(p, false, false)) return AUD_EINVAL;
    *bytes = 4 * scan_space(p, scan_route_of(p, gradients != 0), gradients != 0).all();
    return AUD_OK;
}

int aud_scan_kept_floats(const aud_scan_params* p, int64_t* floats) {
    if (!floats || scan_bad(p, false, false)) return AUD_EINVAL;
    *floats = int64_t(p->n_items) * scan_tiles(p) * p->states * p->channels;
    return AUD_OK;
}

int aud_scan_batch_dev(aud_ctx* c, const aud_scan_params* p, const void* u, const void* delta, const float* A, const void* B,
                       const void* C, const float* D, const void* z, const float* delta_bias, const float* state,
                       const int32_t* lengths, void* y, float* state_out, float* kept, void* workspace, int64_t workspace_bytes,
                       void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = scan_bad(p, z != nullptr, false)) return fail(c, AUD_EINVAL, why);
    if (p->n_items == 0) return AUD_OK;
    const int e = elem_bytes(p->dtype);
    const int64_t bl = int64_t(p->n_items) * p->steps, n = bl * p->channels, ns = int64_t(p->n_items) * p->channels * p->states;
    if ((n && (!u || !delta || !B || !C || !y)) || !A) return fail(c, AUD_EINVAL, "null buffer");
    const int64_t ni = p->n_items, l = p->steps, gn = int64_t(p->groups) * p->states;
    const Input in[] = {{u, ni, l, p->channels, p->u_item, p->u_row}, {delta, ni, l, p->channels, p->delta_item, p->delta_row},
                        {z, ni, l, p->channels, p->z_item, p->z_row}, {B, ni, l, gn, p->b_item, p->b_row}, {C, ni, l, gn, p->c_item, p->c_row}};
    for (const Input& i : in)
        if (!i.aligned(e, e)) return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    if (!at(y, e) || !at(A, 4) || !at(D, 4) || !at(delta_bias, 4) || !at(state, 4) || !at(state_out, 4) || !at(kept, 4) || !at(lengths, 4))
        return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    const aud::ScanRoute r = scan_route_of(p, false);
    int64_t need = 0, kf = 0;
    (void)aud_scan_workspace_bytes(p, 0, &need);
    (void)aud_scan_kept_floats(p, &kf);
    if (int rc = workspace_ok(c, workspace, workspace_bytes, need)) return rc;
    const int64_t ch = 4 * int64_t(p->channels);
    const Range outs[] = {{y, n * e}, {state_out, 4 * ns}, {kept, 4 * kf}, {workspace, need}};
    const Range ins[] = {{u, in[0].span(e)}, {delta, in[1].span(e)}, {z, z ? in[2].span(e) : 0}, {B, in[3].span(e)}, {C, in[4].span(e)},
                         {A, ch * p->states}, {D, ch}, {delta_bias, ch}, {lengths, 4 * ni}, {state == state_out ? nullptr : state, 4 * ns}};
    if (clash(outs, 4, ins, 10)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    if (ni * r.chunks > kMaxGrid / (int64_t(r.blocks) * p->groups) || ns > kMaxGrid * 64 || scan_space(p, r, false).table > kMaxGrid * 256)
        return fail(c, AUD_EINVAL, "tensor too large for one call");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    aud::ScanArgs a{};
    fill_scan(p, r, &a);
    a.u = u, a.delta = delta, a.z = z, a.Bm = B, a.Cm = C, a.A = A, a.D = D, a.delta_bias = delta_bias, a.state = state, a.lengths = lengths;
    a.y = y, a.state_out = state_out, a.kept = kept, a.table = static_cast<float*>(workspace), a.sums = a.table + scan_space(p, r, false).table;
    if (p->steps == 1) {
        AUD_HIP(c, aud::launch_scan_step(a, p->dtype, static_cast<hipStream_t>(stream)));
        return AUD_OK;
    }
    const bool aligned = in[0].aligned(4 * e, e) && in[1].aligned(4 * e, e) && in[2].aligned(4 * e, e) && at(y, 4 * e);
    AUD_HIP(c, aud::launch_scan(a, r, p->dtype, aligned, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

int aud_scan_grad_dev(aud_ctx* c, const aud_scan_params* p, const void* dy, const void* u, const void* delta, const float* A,
                      const void* B, const void* C, const float* D, const void* z, const float* delta_bias, const int32_t* lengths,
                      const float* kept, const float* dstate_out, void* du, void* ddelta, float* dA, void* dB, void* dC, float* dD,
                      void* dz, float* ddelta_bias, float* dstate, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return AUD_EINVAL;
    if (const char* why = scan_bad(p, z != nullptr, true)) return fail(c, AUD_EINVAL, why);
    const int e = elem_bytes(p->dtype);
    const int64_t ni = p->n_items, l = p->steps, gn = int64_t(p->groups) * p->states, n = ni * l * p->channels;
    const int64_t ns = ni * p->channels * p->states, nbc = ni * l * gn, ch = 4 * int64_t(p->channels);
    if (!A || !dA) return fail(c, AUD_EINVAL, "null buffer");
    if (n && (!dy || !u || !delta || !B || !C || !kept || !du || !ddelta || !dB || !dC)) return fail(c, AUD_EINVAL, "null buffer");
    if (n && (z != nullptr) != (dz != nullptr)) return fail(c, AUD_EINVAL, "dz is wanted where z is given, and only there");
    const Input in[] = {{u, ni, l, p->channels, p->u_item, p->u_row}, {delta, ni, l, p->channels, p->delta_item, p->delta_row},
                        {z, ni, l, p->channels, p->z_item, p->z_row}, {dy, ni, l, p->channels, p->dy_item, p->dy_row},
                        {B, ni, l, gn, p->b_item, p->b_row}, {C, ni, l, gn, p->c_item, p->c_row}};
    for (const Input& i : in)
        if (!i.aligned(e, e)) return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    const void* typed[] = {du, ddelta, dz, dB, dC};
    for (const void* q : typed)
        if (!at(q, e)) return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    const void* floats[] = {A, D, delta_bias, lengths, kept, dstate_out, dA, dD, ddelta_bias, dstate};
    for (const void* q : floats)
        if (!at(q, 4)) return fail(c, AUD_EINVAL, "pointer not aligned to its type");
    const aud::ScanRoute r = scan_route_of(p, true);
    int64_t need = 0, kf = 0;
    (void)aud_scan_workspace_bytes(p, 1, &need);
    (void)aud_scan_kept_floats(p, &kf);
    if (int rc = workspace_ok(c, workspace, workspace_bytes, need)) return rc;
    const Range outs[] = {{du, n * e}, {ddelta, n * e}, {dz, n * e}, {dB, nbc * e}, {dC, nbc * e}, {dA, ch * p->states}, {dD, ch},
                          {ddelta_bias, ch}, {dstate, 4 * ns}, {workspace, need}};
    const Range ins[] = {{u, in[0].span(e)}, {delta, in[1].span(e)}, {z, z ? in[2].span(e) : 0}, {dy, in[3].span(e)}, {B, in[4].span(e)},
                         {C, in[5].span(e)}, {A, ch * p->states}, {D, ch}, {delta_bias, ch}, {lengths, 4 * ni}, {kept, 4 * kf}, {dstate_out, 4 * ns}};
    if (clash(outs, 10, ins, 12)) return fail(c, AUD_EINVAL, "an output overlaps another buffer");
    const OnDevice device(c);
    AUD_HIP(c, device.err);
    if (ni == 0) {  // sums over nothing
        AUD_HIP(c, aud::launch_column_sums(nullptr, 0, p->channels, p->states, 2, dA, dD, ddelta_bias, static_cast<hipStream_t>(stream)));
        return AUD_OK;
    }
    if (ni * r.chunks > kMaxGrid / (int64_t(r.blocks) * p->groups) || ns > kMaxGrid * 64 || nbc > kMaxGrid * 64 ||
        scan_space(p, r, true).table > kMaxGrid * 256)
        return fail(c, AUD_EINVAL, "tensor too large for one call");
    const ScanSpace s = scan_space(p, r, true);
    aud::ScanArgs a{};
    fill_scan(p, r, &a);
    a.u = u, a.delta = delta, a.z = z, a.dy = dy, a.Bm = B, a.Cm = C, a.A = A, a.D = D, a.delta_bias = delta_bias, a.lengths = lengths;
    a.kept = const_cast<float*>(kept);  // (only read)
    a.dstate_out = dstate_out, a.du = du, a.ddelta = ddelta, a.dz = dz, a.dB = dB, a.dC = dC;
    a.dA = dA, a.dD = dD, a.ddelta_bias = ddelta_bias, a.dstate = dstate;
    a.table = static_cast<float*>(workspace);
    a.sums = a.table + s.table;
    a.part_bc = a.sums + s.sums;
    a.part = a.part_bc + s.bc;
    const bool aligned = in[0].aligned(4 * e, e) && in[1].aligned(4 * e, e) && in[2].aligned(4 * e, e) && in[3].aligned(4 * e, e) &&
                         at(du, 4 * e) && at(ddelta, 4 * e) && at(dz, 4 * e);
    AUD_HIP(c, aud::launch_scan_grad(a, r, p->dtype, aligned, static_cast<hipStream_t>(stream)));
    return AUD_OK;
}

}  // extern "C"
