// Host side of the operators whose kernels are shorter than it: the autograd nodes of attention with a relative position bias and
// of gated residual norms, and the tensor lists of gradient norm and clipping. A node allocates, makes the calls of
// include/mia_hip.h on the current stream and hands torch the gradients, as the torch.autograd.Functions of ops.py do. In C++
// because the kernels of a head take about 50 us and its host side in Python took 120: one pass forward and backward of
// attention over 16 x 100 tokens in 8 heads, fp32, 122 -> 68 us; a residual of 361 x 2304, fp32, 124 -> 81; clipping 430 tensors
// 136 -> 41. Arguments are checked by the Python functions that call this (relpos.py, block_norm.py, optim.py).
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <mutex>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include "../../include/mia_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char* name) {
    if (rc) throw Refused(std::string(name) + " failed (" + std::to_string(rc) + "): " + mia_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MIA_BF16 : MIA_F32; }
bool aligned(const Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15) == 0; }
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor dense_aligned(const Tensor& t) {
    Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}
const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const float* cfloats(const Tensor& t) { return static_cast<const float*>(cptr(t)); }
void* ptr(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* floats(Tensor& t) { return static_cast<float*>(ptr(t)); }

template <typename... T>
bool recorded(const T&... t) {
    return c10::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// Under create_graph=True the results would be taken for constants.
void first_derivative_only(const char* name) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), name, " has no second derivative (create_graph=True)");
}

// The kernels see values alone: a result would be a constant to forward-mode differentiation. Tangents exist inside a dual level
// only, so that is asked first (tensor by tensor the question takes 12 us for the 430 gradients of a model).
bool in_dual_level() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name, " has no forward-mode derivative");
}
template <typename... T>
void no_tangents(const char* name, const T&... t) {
    if (in_dual_level()) (no_tangent(name, t), ...);
}

// A tracer sees the allocation of a result and not the kernels that fill it: its program would return memory as it was.
void not_traced(const char* name) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), name,
                " cannot be traced (torch.jit.trace, make_fx, torch.export): its kernels would be missing from the program");
}

// A saved tensor as it comes back. Hooks may return the values in another layout (save_on_cpu does so for a view that is not
// dense), so nothing about addresses, strides or alignment is taken over from the forward; shape, type and device have to be the same.
Tensor restored(const Tensor& t, at::IntArrayRef shape, at::ScalarType type, at::Device device, const char* name) {
    TORCH_CHECK(t.defined() && t.sizes() == shape && t.scalar_type() == type && t.device() == device && t.layout() == at::kStrided, name,
                ": a saved tensor came back from its hooks as ", t.defined() ? c10::str(t.scalar_type(), t.sizes(), " on ", t.device()) : "nothing",
                " (was ", type, shape, " on ", device, ")");
    return t;
}

// ------------------------------------------------------------------------------------------------
// attention with a relative position bias
// ------------------------------------------------------------------------------------------------
struct Attention {
    int B, heads, Lq, Lk, D, height, width, buckets, q_start;
    float scale, pdrop;
    unsigned long long seed;
    const unsigned long long* seed_offset;
    at::ScalarType type, mask_type;
    at::Device device = at::kCPU;
    bool packed, empty;

    std::vector<int64_t> query_shape() const { return packed ? std::vector<int64_t>{B, Lq, 3, heads, D} : std::vector<int64_t>{B, Lq, heads, D}; }
    std::vector<int64_t> key_shape() const { return {B, Lk, heads, D}; }
};

// (batch, token, head) strides in elements; one of a dimension of length one does not matter
void strides_of(const Tensor& t, long long* st) {
    for (int i = 0; i < 3; ++i) st[i] = t.size(i) == 1 ? 0 : t.stride(i);
}

// The tensor itself when the kernels can read it where it lies (head elements contiguous, rows at multiples of 16 bytes), else
// a contiguous copy
Tensor readable(const Tensor& t, long long* st) {
    const long long per = 16 / t.element_size();
    strides_of(t, st);
    if ((t.stride(3) == 1 || t.size(3) == 1) && st[0] % per == 0 && st[1] % per == 0 && st[2] % per == 0 && st[1] < 1ll << 24 && aligned(t)) return t;
    const Tensor c = dense_aligned(t);
    strides_of(c, st);
    return c;
}

// addresses and strides of q, k and v inside a packed [B, L, 3, heads, D] tensor
void packed_rows(const Tensor& t, const char** at, long long* st) {
    for (int i = 0; i < 3; ++i) {
        at[i] = static_cast<const char*>(t.const_data_ptr()) + i * t.stride(2) * t.element_size();
        st[3 * i] = t.stride(0);
        st[3 * i + 1] = t.stride(1);
        st[3 * i + 2] = t.stride(3);
    }
}

struct RelPosAttentionBackward : torch::autograd::Node {
    Attention a;
    SavedVariable q, k, v, bias, mask, out, low, stat;
    Tensor order, start;
    std::array<int64_t, 2> table;
    int64_t offsets;
    bool masked;

    std::string name() const override { return "RelPosAttentionBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* s : {&q, &k, &v, &bias, &mask, &out, &low, &stat}) s->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        first_derivative_only("relpos_attention");
        variable_list got(4);
        if (!grads[0].defined()) return got;
        const c10::DeviceGuard guard(a.device);
        const auto options = at::TensorOptions().device(a.device).dtype(a.type), f32 = options.dtype(at::kFloat);
        const auto query_shape = a.query_shape(), key_shape = a.key_shape();
        const bool want = task_should_compute_output(3);
        if (a.empty) {
            got[0] = at::zeros(query_shape, options);
            if (!a.packed) got[1] = at::zeros(key_shape, options), got[2] = at::zeros(key_shape, options);
            if (want) got[3] = at::zeros(table, f32);
            return got;
        }
        const auto back = [this](const Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
            return restored(t, shape, type, a.device, "relpos_attention");
        };
        const std::array<int64_t, 4> rows = {a.B, a.Lq, a.heads, a.D};
        Tensor q_ = back(q.unpack(), query_shape, a.type), k_ = k.unpack(), v_ = v.unpack(), mask_ = mask.unpack(), low_ = low.unpack();
        const Tensor bias_ = dense(back(bias.unpack(), {a.heads, offsets}, at::kFloat));
        const Tensor stat_ = dense_aligned(back(stat.unpack(), {a.B, a.heads, a.Lq, 2}, at::kFloat));
        const Tensor out_ = dense_aligned(back(out.unpack(shared_from_this()), rows, a.type));
        if (a.type == at::kBFloat16) low_ = dense_aligned(back(low_, rows, a.type));
        if (masked) mask_ = dense(back(mask_, {a.B, a.Lk}, a.mask_type));
        const Tensor dout = dense_aligned(grads[0]);
        const char* in[3];
        char* grad[3];
        long long strides[9], gst[9];
        got[0] = at::empty(query_shape, options);
        if (a.packed) {
            q_ = dense_aligned(q_);
            packed_rows(q_, in, strides);
            const char* at[3];
            packed_rows(got[0], at, gst);
            for (int i = 0; i < 3; ++i) grad[i] = const_cast<char*>(at[i]);
        } else {
            got[1] = at::empty(key_shape, options);
            got[2] = at::empty(key_shape, options);
            q_ = readable(q_, strides), k_ = readable(back(k_, key_shape, a.type), strides + 3), v_ = readable(back(v_, key_shape, a.type), strides + 6);
            const Tensor* of[3] = {&q_, &k_, &v_};
            for (int i = 0; i < 3; ++i) {
                in[i] = static_cast<const char*>(of[i]->const_data_ptr());
                grad[i] = static_cast<char*>(got[i].mutable_data_ptr());
                for (int d = 0; d < 3; ++d) gst[3 * i + d] = got[i].stride(d);
            }
        }
        if (want) got[3] = at::empty(table, f32);
        const int dt = dtype_of(q_);
        const long long n = mia_relpos_bwd_ws_floats(dt, a.B, a.heads, a.Lq, a.Lk, a.D, a.height, a.width, want);
        Tensor ws = at::empty({n}, f32);
        check(mia_relpos_bwd(dt, in[0], in[1], in[2], strides, dout.const_data_ptr(), out_.const_data_ptr(), cptr(low_), cfloats(stat_), a.B,
                             a.heads, a.Lq, a.Lk, a.D, cfloats(bias_), a.height, a.width, a.q_start, static_cast<const uint8_t*>(cptr(mask_)), a.scale,
                             a.pdrop, a.seed, a.seed_offset, static_cast<const int*>(cptr(order)), static_cast<const int*>(cptr(start)), a.buckets,
                             floats(ws), n, grad[0], grad[1], grad[2], gst, floats(got[3]), stream_of(q_)),
              "mia_relpos_bwd");
        return got;
    }
};

// q, k, v or one packed tensor in the place of q. What the backward needs is written only where autograd records the call.
Tensor relpos(Tensor q, const Maybe& k_in, const Maybe& v_in, const Tensor& table_in, const Tensor& index, const Tensor& order, const Tensor& start,
              const Maybe& mask_in, int height, int width, int buckets, double scale, int q_start, double pdrop, unsigned long long seed,
              unsigned long long seed_offset) {
    Tensor k = or_none(k_in), v = or_none(v_in), mask = or_none(mask_in), out;
    not_traced("relpos_attention");
    no_tangents("relpos_attention", q, k, v, table_in);
    std::shared_ptr<RelPosAttentionBackward> node;
    if (recorded(q, k, v, table_in)) {
        node = std::shared_ptr<RelPosAttentionBackward>(new RelPosAttentionBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, v, table_in));
    }
    {
        const at::NoGradGuard quiet;
        const c10::DeviceGuard guard(q.device());
        Attention a = {};
        a.packed = !k.defined();
        a.B = q.size(0), a.Lq = q.size(1), a.Lk = a.packed ? a.Lq : k.size(1), a.heads = q.size(a.packed ? 3 : 2), a.D = q.size(a.packed ? 4 : 3);
        a.height = height, a.width = width, a.buckets = buckets, a.q_start = q_start;
        a.scale = (float)scale, a.pdrop = (float)pdrop, a.seed = seed;
        a.seed_offset = reinterpret_cast<const unsigned long long*>(seed_offset);
        a.type = q.scalar_type(), a.device = q.device();
        a.empty = a.B == 0 || a.Lq == 0 || a.Lk == 0 || a.heads == 0;
        const auto f32 = q.options().dtype(at::kFloat);
        const std::array<int64_t, 4> rows = {a.B, a.Lq, a.heads, a.D};
        Tensor bias, low, stat;
        if (a.empty) {
            out = at::zeros(rows, q.options());
        } else {
            const char* in[3];
            long long strides[9];
            if (a.packed) {
                q = dense_aligned(q);
                packed_rows(q, in, strides);
            } else {
                q = readable(q, strides), k = readable(k, strides + 3), v = readable(v, strides + 6);
                const Tensor* of[3] = {&q, &k, &v};
                for (int i = 0; i < 3; ++i) in[i] = static_cast<const char*>(of[i]->const_data_ptr());
            }
            out = at::empty(rows, q.options());
            bias = at::empty({a.heads, index.numel()}, f32);
            if (node) {
                stat = at::empty({a.B, a.heads, a.Lq, 2}, f32);
                if (q.scalar_type() == at::kBFloat16) low = at::empty(rows, q.options());
            }
            const Tensor table = table_in.contiguous();
            mask = dense(mask);
            const int dt = dtype_of(q);
            const long long n = mia_relpos_fwd_ws_floats(dt, a.B, a.heads, a.Lq, a.Lk, a.D);
            Tensor ws = n ? at::empty({n}, f32) : Tensor();
            void* stream = stream_of(q);
            check(mia_relpos_bias(cfloats(table), static_cast<const int*>(cptr(index)), height, width, a.heads, a.scale, floats(bias), stream), "mia_relpos_bias");
            check(mia_relpos_fwd(dt, in[0], in[1], in[2], strides, a.B, a.heads, a.Lq, a.Lk, a.D, floats(bias), height, width, q_start,
                                 static_cast<const uint8_t*>(cptr(mask)), a.scale, a.pdrop, seed, a.seed_offset, floats(ws), n, ptr(out), ptr(low),
                                 floats(stat), stream),
                  "mia_relpos_fwd");
        }
        if (node) {
            a.mask_type = mask.defined() ? mask.scalar_type() : at::kBool;
            node->a = a, node->offsets = index.numel(), node->masked = mask.defined();
            node->order = order, node->start = start;
            node->table = {table_in.size(0), table_in.size(1)};
            node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->v = SavedVariable(v, false);
            node->bias = SavedVariable(bias, false), node->mask = SavedVariable(mask, false);
            node->low = SavedVariable(low, false), node->stat = SavedVariable(stat, false);
        }
    }
    if (node) {
        torch::autograd::set_history(out, node);
        if (!node->a.empty) node->out = SavedVariable(out, true);
    }
    return out;
}

// ------------------------------------------------------------------------------------------------
// gated residual norms
// ------------------------------------------------------------------------------------------------
struct GatedResidualNormBackward : torch::autograd::Node {
    SavedVariable x, f, stats, parameter[6];   // scale, gate, w1, b1, w2, b2
    bool has[6];
    at::ScalarType type;
    at::Device device = at::kCPU;
    std::vector<int64_t> shape;
    int images, C, post, pre;
    long long rows;   // of an image

    std::string name() const override { return "GatedResidualNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(), f.reset_data(), stats.reset_data();
        for (SavedVariable& p : parameter) p.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        first_derivative_only("gated_residual_norm");
        variable_list got(8);
        Tensor dy = grads[0], dz = pre ? grads[1] : Tensor();
        if (!dy.defined() && !dz.defined()) return got;
        const c10::DeviceGuard guard(device);
        const auto options = at::TensorOptions().device(device).dtype(type), f32 = options.dtype(at::kFloat);
        const auto back = [this](const Tensor& t, at::IntArrayRef of, at::ScalarType as) { return restored(t, of, as, device, "gated_residual_norm"); };
        const std::vector<int64_t> gate = {images, C}, vector = {C};
        got[0] = at::empty(shape, options), got[1] = at::empty(shape, options);
        for (int i = 0; i < 6; ++i)
            if (has[i] && task_should_compute_output(2 + i)) got[2 + i] = rows ? at::empty(i == 1 ? gate : vector, f32) : at::zeros(i == 1 ? gate : vector, f32);
        if (!rows) return got;
        // rows that can be read 16 bytes at a time are: their layout, and with it the order of the sums, does not hang on a hook
        const auto rows_of = C % (type == at::kBFloat16 ? 8 : 4) ? dense : dense_aligned;
        const Tensor x_ = rows_of(back(x.unpack(), shape, type)), f_ = rows_of(back(f.unpack(), shape, type));
        const Tensor stats_ = dense_aligned(back(stats.unpack(), {images * rows, 4}, at::kFloat));
        Tensor p[6];
        for (int i = 0; i < 6; ++i)
            if (has[i]) p[i] = rows_of(back(parameter[i].unpack(), i == 1 ? gate : vector, at::kFloat));
        dy = dense(dy), dz = dense(dz);
        const long long n = mia_blocknorm_ws_floats(images, rows, C, p[1].defined());
        Tensor ws = at::empty({n}, f32);
        check(mia_blocknorm_bwd(dtype_of(x_), cptr(dy), cptr(dz), cptr(x_), cptr(f_), cfloats(stats_), images, rows, C, cfloats(p[0]), cfloats(p[1]),
                                post, cfloats(p[2]), cfloats(p[3]), pre, cfloats(p[4]), floats(ws), n, ptr(got[0]), ptr(got[1]), floats(got[2]),
                                floats(got[3]), floats(got[4]), floats(got[5]), floats(got[6]), floats(got[7]), stream_of(x_)),
              "mia_blocknorm_bwd");
        return got;
    }
};

std::tuple<Tensor, Maybe> residual(const Tensor& x_in, const Tensor& f_in, const Maybe& scale, const Maybe& gate, const Maybe& w1, const Maybe& b1,
                                   const Maybe& w2, const Maybe& b2, int post, int pre, double eps) {
    const Maybe* maybe[6] = {&scale, &gate, &w1, &b1, &w2, &b2};
    Tensor p[6], y, z;
    for (int i = 0; i < 6; ++i) p[i] = or_none(*maybe[i]);
    not_traced("gated_residual_norm");
    no_tangents("gated_residual_norm", x_in, f_in, p[0], p[1], p[2], p[3], p[4], p[5]);
    std::shared_ptr<GatedResidualNormBackward> node;
    if (recorded(x_in, f_in, p[0], p[1], p[2], p[3], p[4], p[5])) {
        node = std::shared_ptr<GatedResidualNormBackward>(new GatedResidualNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, f_in, p[0], p[1], p[2], p[3], p[4], p[5]));
    }
    {
        const at::NoGradGuard quiet;
        const c10::DeviceGuard guard(x_in.device());
        const Tensor x = x_in.contiguous(), f = f_in.contiguous();
        for (Tensor& t : p) t = dense(t);
        const int C = (int)x.size(-1), images = p[1].defined() ? (int)p[1].size(0) : 1;
        const long long rows = x.numel() ? x.numel() / ((long long)images * C) : 0;
        y = at::empty_like(x);
        if (pre) z = at::empty_like(x);
        Tensor stats = node ? at::empty({images * rows, 4}, x.options().dtype(at::kFloat)) : Tensor();
        if (rows)
            check(mia_blocknorm_fwd(dtype_of(x), cptr(x), cptr(f), images, rows, C, cfloats(p[0]), cfloats(p[1]), post, cfloats(p[2]), cfloats(p[3]), pre,
                                    cfloats(p[4]), cfloats(p[5]), (float)eps, ptr(y), ptr(z), floats(stats), stream_of(x)),
                  "mia_blocknorm_fwd");
        if (node) {
            node->images = images, node->rows = rows, node->C = C, node->post = post, node->pre = pre;
            node->type = x.scalar_type(), node->device = x.device(), node->shape = x.sizes().vec();
            node->x = SavedVariable(x, false), node->f = SavedVariable(f, false), node->stats = SavedVariable(stats, false);
            for (int i = 0; i < 6; ++i) node->parameter[i] = SavedVariable(p[i], false), node->has[i] = p[i].defined();
        }
    }
    if (node) {
        torch::autograd::set_history(y, node);
        if (pre) torch::autograd::set_history(z, node);
    }
    return {y, pre ? Maybe(z) : std::nullopt};
}

// ------------------------------------------------------------------------------------------------
// gradient norm and clipping: reading the addresses, sizes and types of a few hundred tensors is most of the work
// ------------------------------------------------------------------------------------------------
bool dense_layout(const Tensor& t) {   // the elements fill one run of memory in some order
    if (t.layout() != at::kStrided) throw py::type_error("gradients are dense tensors");
    return t.is_non_overlapping_and_dense();
}

bool all_dense(const std::vector<Tensor>& grads) { return std::all_of(grads.begin(), grads.end(), dense_layout); }

struct GradTable {
    std::vector<const void*> at;
    std::vector<int> dtypes;
    std::vector<long long> sizes;
    Tensor ws, out;   // out: norm and factor

    explicit GradTable(const std::vector<Tensor>& grads) {
        not_traced("gradient norm and clipping");
        const bool dual = in_dual_level();
        for (const Tensor& g : grads) {
            if (dual) no_tangent("gradient norm and clipping", g);
            if (!g.is_cuda() || g.device() != grads[0].device())
                throw std::runtime_error("gradient norm and clipping need their tensors on one MI355X device; there is no CPU path");
            if (g.scalar_type() != at::kFloat && g.scalar_type() != at::kBFloat16)
                throw py::type_error(std::string("gradients are fp32 or bf16 (got ") + toString(g.scalar_type()) + ")");
            at.push_back(g.const_data_ptr());
            dtypes.push_back(dtype_of(g));
            sizes.push_back(g.numel());
        }
        const auto here = at::TensorOptions().device(grads[0].device());
        ws = at::empty({mia_grad_norm_ws_doubles(count(), sizes.data())}, here.dtype(at::kDouble));
        out = at::empty({2}, here.dtype(at::kFloat));
    }
    int count() const { return (int)at.size(); }
};

Tensor grad_norm(std::vector<Tensor> grads) {
    const at::NoGradGuard quiet;
    for (Tensor& g : grads)
        if (!dense_layout(g)) g = g.contiguous();
    const c10::OptionalDeviceGuard guard(at::device_of(grads[0]));
    GradTable t(grads);
    check(mia_grad_norm(t.count(), t.at.data(), t.dtypes.data(), t.sizes.data(), 1.0, 0.0, static_cast<double*>(ptr(t.ws)), t.ws.numel(), floats(t.out),
                        stream_of(t.ws)),
          "mia_grad_norm");
    return t.out.select(0, 0);
}

Tensor grad_clip(const std::vector<Tensor>& grads, double max_norm) {
    const at::NoGradGuard quiet;
    for (const Tensor& g : grads)
        if (!dense_layout(g))
            throw py::value_error("clip_grads_ scales in place and needs dense tensors (got strides " + c10::str(g.strides()) + " for " + c10::str(g.sizes()) + ")");
    const c10::OptionalDeviceGuard guard(at::device_of(grads[0]));
    GradTable t(grads);
    std::vector<std::pair<const char*, const char*>> each;   // first and last byte; in this order any overlap shows between neighbours
    for (int i = 0; i < t.count(); ++i) {
        const char* p = static_cast<const char*>(t.at[i]);
        if (t.sizes[i]) each.emplace_back(p, p + t.sizes[i] * grads[i].element_size() - 1);
    }
    std::sort(each.begin(), each.end());
    for (size_t i = 1; i < each.size(); ++i)
        if (each[i].first <= each[i - 1].second)
            throw py::value_error(each[i] == each[i - 1] ? "a tensor is listed twice: it would be scaled twice"
                                                         : "two tensors overlap: their common elements would be scaled twice");
    check(mia_grad_clip(t.count(), t.at.data(), t.dtypes.data(), t.sizes.data(), max_norm, static_cast<double*>(ptr(t.ws)), t.ws.numel(), floats(t.out),
                        stream_of(t.ws)),
          "mia_grad_clip");
    for (const Tensor& g : grads)
        if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();   // written in place
    return t.out.select(0, 0);
}

// Whether AdamW's kernel can take every parameter and its gradient as they are: dense fp32 on the device
bool update_ready(const std::vector<Tensor>& params) {
    return std::all_of(params.begin(), params.end(), [](const Tensor& p) {
        const Tensor& g = p.grad();
        return g.defined() && p.is_cuda() && g.is_cuda() && p.scalar_type() == at::kFloat && g.scalar_type() == at::kFloat &&
               g.layout() == at::kStrided && p.is_contiguous() && g.is_contiguous();
    });
}

PyObject* refusal = nullptr;   // the library's exception class

}  // namespace

PYBIND11_MODULE(_mia_autograd, m) {
    m.def("digest", []() { return MIA_HEADER_DIGEST; }, "Digest of the prototypes that this module was compiled against.");
    m.def("bind", [](py::object error) { refusal = error.release().ptr(); });
    m.def("relpos", &relpos, py::call_guard<py::gil_scoped_release>());
    m.def("residual", &residual, py::call_guard<py::gil_scoped_release>());
    m.def("all_dense", &all_dense);
    m.def("update_ready", &update_ready);
    m.def("grad_norm", &grad_norm, py::call_guard<py::gil_scoped_release>());
    m.def("grad_clip", &grad_clip, py::call_guard<py::gil_scoped_release>());
    py::register_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const Refused& r) {
            PyErr_SetString(refusal ? refusal : PyExc_RuntimeError, r.what());
        }
    });
}
