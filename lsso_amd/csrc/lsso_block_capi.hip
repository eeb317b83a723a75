// C ABI of the operators around the mixer (token embedding, gated feed-forward
// block, residual dropout):
// host-side validation, workspace planning and stream-ordered launches, as in
// lsso_capi.hip.  No exception leaves these entries: nothing here allocates.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "lsso_hip.h"
#include "lsso_internal.h"

namespace {

using lsso_hip::report;
using lsso_hip::report_hip;

bool value_type(int type) { return type == LSSO_HIP_F16 || type == LSSO_HIP_BF16 || type == LSSO_HIP_F32; }
bool aligned(const void* pointer, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(pointer) % bytes == 0; }
uintptr_t type_bytes(int type) { return type == LSSO_HIP_F32 ? 4 : 2; }

constexpr int64_t kMostIds = 0x7fffffff;
constexpr int64_t kMostFeatures = 1 << 22;

int check_embedding(const void* tokens, int token_bytes, int64_t count, int64_t vocabulary, int64_t dim) {
    if (count < 0 || vocabulary <= 0 || dim <= 0) {
        return report(LSSO_HIP_EINVAL, "count must not be negative, vocabulary and dim must be positive");
    }
    if (count > kMostIds || vocabulary > kMostIds - 1 || dim > kMostFeatures) {
        return report(LSSO_HIP_EUNSUPPORTED, "the embedding takes fewer than 2^31 tokens and rows of up to 2^22 features");
    }
    if (token_bytes != 4 && token_bytes != 8) {
        return report(LSSO_HIP_EINVAL, "tokens must be int32 or int64");
    }
    if (count > 0 && (tokens == nullptr || !aligned(tokens, token_bytes))) {
        return report(LSSO_HIP_EINVAL, "tokens must not be NULL and be aligned to their type");
    }
    return LSSO_HIP_OK;
}

size_t round256(size_t bytes) { return (bytes + 255) & ~static_cast<size_t>(255); }
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
// Bytes per row of what fine factors keep beside their upper 16 bits.
int64_t lower_pitch(const lsso_hip_feed_forward_shape& s) {
    return (s.hidden + 31) / 32 * (s.dtype == LSSO_HIP_BF16 ? 32 : 64);
}

// Rows whose pieces the product's loads can address: 16-byte pieces, and 256
// rows within a buffer's 2^31 bytes.
bool whole_rows(int64_t columns, int64_t stride) {
    return columns % 8 == 0 && stride % 8 == 0 && stride < (1 << 21);
}

int check_feed_forward(const lsso_hip_feed_forward_shape* s) {
    if (s == nullptr) {
        return report(LSSO_HIP_EINVAL, "shape must not be NULL");
    }
    if (s->rows < 0 || s->in_features <= 0 || s->hidden <= 0 || s->out_features <= 0) {
        return report(LSSO_HIP_EINVAL, "rows must not be negative, features and hidden must be positive");
    }
    constexpr int64_t most = 1 << 20;
    if (s->rows > kMostIds || s->in_features > most || s->hidden > most || s->out_features > most) {
        return report(LSSO_HIP_EUNSUPPORTED,
                      "the feed-forward block takes fewer than 2^31 rows and widths of up to 2^20");
    }
    if (s->dtype != LSSO_HIP_F16 && s->dtype != LSSO_HIP_BF16) {
        return report(LSSO_HIP_EUNSUPPORTED, "the feed-forward block takes float16 or bfloat16 activations");
    }
    if (s->weight_type != s->dtype && s->weight_type != LSSO_HIP_F32) {
        return report(LSSO_HIP_EUNSUPPORTED, "the weights must have the activations' type or float32");
    }
    if (s->activation != LSSO_HIP_SILU && s->activation != LSSO_HIP_GELU) {
        return report(LSSO_HIP_EUNSUPPORTED, "activation must be LSSO_HIP_SILU or LSSO_HIP_GELU");
    }
    if (s->fine_factors != 0 && s->fine_factors != 1) {
        return report(LSSO_HIP_EINVAL, "fine_factors must be 0 or 1");
    }
    if (s->x_stride < s->in_features) {
        return report(LSSO_HIP_EINVAL, "x_stride must be at least in_features");
    }
    return LSSO_HIP_OK;
}

// Workspace and argument blocks of both directions; pointers are offsets into
// the workspace until bind() adds its address.
struct FeedForwardPlan {
    lsso_hip::FeedForwardPack pack{};
    lsso_hip::FeedForwardArgs args{};
    lsso_hip::FeedForwardProduct product{};
    lsso_hip::FeedForwardWeights weights{};
    size_t bytes = 0;

    size_t take(size_t size) {
        const size_t at = bytes;
        bytes += round256(size);
        return at;
    }
};

// The operand `from` [rows, columns] as 16-bit rows of whole pieces: itself, or
// a copy in the workspace.
struct Packed {
    bool copied = false;
    size_t offset = 0;
    int64_t stride = 0;
};

Packed place(FeedForwardPlan* plan, int64_t rows, int64_t columns, int64_t stride, bool wide) {
    Packed p;
    p.copied = wide || !whole_rows(columns, stride);
    p.stride = p.copied ? round8(columns) : stride;
    if (p.copied) {
        p.offset = plan->take(2 * static_cast<size_t>(rows) * static_cast<size_t>(p.stride));
    }
    return p;
}

const uint16_t* bind(FeedForwardPlan* plan, const Packed& p, const void* from, int64_t rows, int64_t columns,
                     int64_t stride, bool wide, char* workspace) {
    if (!p.copied) {
        return static_cast<const uint16_t*>(from);
    }
    uint16_t* to = reinterpret_cast<uint16_t*>(workspace + p.offset);
    plan->pack.matrices[plan->pack.count++] = {from, stride, rows, columns, wide, 0, to, p.stride, 0};
    return to;
}

// The transpose of `from` [rows, columns] as rows of `pitch` values at `to`.
void transpose(FeedForwardPlan* plan, const void* from, int64_t rows, int64_t columns, bool wide, uint16_t* to,
               int64_t pitch) {
    plan->pack.matrices[plan->pack.count++] = {from, columns, rows, columns, wide, 1, to, pitch, 0};
}

struct FeedForwardLayout {
    FeedForwardPlan plan;
    Packed x, gate, up, down, dy;
    size_t h = 0, h_low = 0, partials = 0, grads = 0, weight_partials = 0;
    size_t in_columns = 0, down_columns = 0;   // [gate^T | up^T] [in, 2 pitch], down^T [hidden, out_pitch]
};

void common_args(const lsso_hip_feed_forward_shape& s, lsso_hip::FeedForwardArgs* a) {
    a->type = s.dtype;
    a->activation = s.activation;
    a->rows = s.rows;
    a->hidden = s.hidden;
    a->out_features = s.out_features;
    a->in_pitch = round8(s.in_features);
    a->pitch = round8(s.hidden);
    a->out_pitch = round8(s.out_features);
    a->lower_pitch = lower_pitch(s);
}

// The kept factors: 16 bits of each, and behind all of them the rest of fine ones.
void bind_gates(const lsso_hip_feed_forward_shape& s, void* gates, lsso_hip::FeedForwardArgs* a) {
    a->gates = static_cast<uint16_t*>(gates);
    if (gates != nullptr && s.fine_factors != 0) {
        a->gates_lower = reinterpret_cast<char*>(a->gates + 2 * s.rows * a->pitch);
    }
}

int64_t stages_of(int64_t k) { return (k + 63) / 64; }

FeedForwardLayout forward_layout(const lsso_hip_feed_forward_shape& s, bool training) {
    FeedForwardLayout l;
    common_args(s, &l.plan.args);
    const bool wide = s.weight_type == LSSO_HIP_F32;
    l.x = place(&l.plan, s.rows, s.in_features, s.x_stride, false);
    l.gate = place(&l.plan, s.hidden, s.in_features, s.in_features, wide);
    l.up = place(&l.plan, s.hidden, s.in_features, s.in_features, wide);
    l.down = place(&l.plan, s.out_features, s.hidden, s.hidden, wide);
    const size_t pitch = static_cast<size_t>(l.plan.args.pitch);
    if (!training) {
        l.h = l.plan.take(2 * static_cast<size_t>(s.rows) * pitch);
    }
    if (s.rows <= lsso_hip::kFewRows) {
        l.h_low = l.plan.take(2 * static_cast<size_t>(s.rows) * pitch);
    }
    lsso_hip::FeedForwardProduct& y = l.plan.product;
    lsso_hip::plan_product(s.rows, s.out_features, stages_of(l.plan.args.pitch), &y);
    if (y.splits > 1) {
        l.partials = l.plan.take(4 * static_cast<size_t>(y.splits) * static_cast<size_t>(s.rows) *
                                 static_cast<size_t>(y.partial_pitch));
    }
    return l;
}

// The weight gradients' products in the order gate, up, down.
void weight_products(const lsso_hip_feed_forward_shape& s, const bool (&wanted)[3], FeedForwardPlan* plan) {
    const lsso_hip::FeedForwardArgs& a = plan->args;
    lsso_hip::FeedForwardWeights& w = plan->weights;
    w.type = s.dtype;
    w.rows = s.rows;
    w.count = 0;
    for (int i = 0; i < 3; ++i) {
        if (!wanted[i]) {
            continue;
        }
        lsso_hip::WeightProduct& p = w.products[w.count++];
        p = {};
        if (i < 2) {
            p.p_stride = 2 * a.pitch;
            p.p_columns = a.pitch;
            p.q_columns = a.in_pitch;
            p.out_rows = s.hidden;
            p.partial_pitch = a.in_pitch;
        } else {
            p.p_columns = a.out_pitch;
            p.q_stride = a.pitch;
            p.q_columns = a.pitch;
            p.out_rows = s.out_features;
            p.partial_pitch = a.pitch;
        }
    }
    lsso_hip::plan_weights(&w);
}

FeedForwardLayout backward_layout(const lsso_hip_feed_forward_shape& s, int64_t grad_stride, const bool (&wanted)[3]) {
    FeedForwardLayout l;
    common_args(s, &l.plan.args);
    const lsso_hip::FeedForwardArgs& a = l.plan.args;
    l.x = place(&l.plan, s.rows, s.in_features, s.x_stride, false);
    l.dy = place(&l.plan, s.rows, s.out_features, grad_stride, false);
    l.in_columns = l.plan.take(2 * static_cast<size_t>(s.in_features) * 2 * static_cast<size_t>(a.pitch));
    l.down_columns = l.plan.take(2 * static_cast<size_t>(s.hidden) * static_cast<size_t>(a.out_pitch));
    l.grads = l.plan.take(4 * static_cast<size_t>(s.rows) * static_cast<size_t>(a.pitch));
    lsso_hip::FeedForwardProduct& dx = l.plan.product;
    lsso_hip::plan_product(s.rows, s.in_features, stages_of(2 * a.pitch), &dx);
    if (dx.splits > 1) {
        l.partials = l.plan.take(4 * static_cast<size_t>(dx.splits) * static_cast<size_t>(s.rows) *
                                 static_cast<size_t>(dx.partial_pitch));
    }
    weight_products(s, wanted, &l.plan);
    if (l.plan.weights.count > 0) {
        l.weight_partials = l.plan.take(4 * static_cast<size_t>(l.plan.weights.splits) *
                                        static_cast<size_t>(l.plan.weights.partial_floats));
    }
    return l;
}

}  // namespace

extern "C" {

int lsso_hip_feed_forward_kept(const lsso_hip_feed_forward_shape* shape, size_t* gates, size_t* product) {
    const int status = check_feed_forward(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (gates == nullptr || product == nullptr) {
        return report(LSSO_HIP_EINVAL, "gates and product must not be NULL");
    }
    *product = static_cast<size_t>(shape->rows) * static_cast<size_t>(round8(shape->hidden));
    *gates = 2 * *product;
    if (shape->fine_factors != 0) {
        *gates += static_cast<size_t>(shape->rows) * static_cast<size_t>(lower_pitch(*shape) / 2);
    }
    return LSSO_HIP_OK;
}

int lsso_hip_feed_forward_workspace_bytes(const lsso_hip_feed_forward_shape* shape, int training, size_t* bytes) {
    const int status = check_feed_forward(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (bytes == nullptr) {
        return report(LSSO_HIP_EINVAL, "bytes must not be NULL");
    }
    *bytes = forward_layout(*shape, training != 0).plan.bytes;
    return LSSO_HIP_OK;
}

int lsso_hip_feed_forward(const lsso_hip_feed_forward_shape* shape, const void* x, const void* gate_weight,
                          const void* up_weight, const void* down_weight, const uint8_t* row_mask, void* gates,
                          void* product, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    const int status = check_feed_forward(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if ((gates == nullptr) != (product == nullptr)) {
        return report(LSSO_HIP_EINVAL, "gates and product are given together or not at all");
    }
    const lsso_hip_feed_forward_shape& s = *shape;
    if (s.rows == 0) {
        return LSSO_HIP_OK;
    }
    if (x == nullptr || gate_weight == nullptr || up_weight == nullptr || down_weight == nullptr || y == nullptr) {
        return report(LSSO_HIP_EINVAL, "x, the weights and y must not be NULL");
    }
    if (!aligned(x, 16) || !aligned(gate_weight, 16) || !aligned(up_weight, 16) || !aligned(down_weight, 16) ||
        !aligned(gates, 16) || !aligned(product, 16) || !aligned(y, 2)) {
        return report(LSSO_HIP_EINVAL, "x, the weights, gates and product must be 16-byte aligned");
    }
    FeedForwardLayout l = forward_layout(s, gates != nullptr);
    if (l.plan.bytes > 0 && (workspace == nullptr || workspace_bytes < l.plan.bytes || !aligned(workspace, 256))) {
        return report(LSSO_HIP_EINVAL,
                      "workspace must be 256-byte aligned and of lsso_hip_feed_forward_workspace_bytes()");
    }
    char* ws = static_cast<char*>(workspace);
    const bool wide = s.weight_type == LSSO_HIP_F32;
    lsso_hip::FeedForwardArgs& a = l.plan.args;
    a.x = bind(&l.plan, l.x, x, s.rows, s.in_features, s.x_stride, false, ws);
    a.x_stride = l.x.stride;
    a.gate = bind(&l.plan, l.gate, gate_weight, s.hidden, s.in_features, s.in_features, wide, ws);
    a.up = bind(&l.plan, l.up, up_weight, s.hidden, s.in_features, s.in_features, wide, ws);
    a.down = bind(&l.plan, l.down, down_weight, s.out_features, s.hidden, s.hidden, wide, ws);
    a.row_mask = row_mask;
    bind_gates(s, gates, &a);
    a.h = product != nullptr ? static_cast<uint16_t*>(product) : reinterpret_cast<uint16_t*>(ws + l.h);
    const bool few = s.rows <= lsso_hip::kFewRows;
    a.h_low = few ? reinterpret_cast<uint16_t*>(ws + l.h_low) : nullptr;
    lsso_hip::FeedForwardProduct& p = l.plan.product;
    p.type = s.dtype;
    p.p = a.h;
    p.p_low = a.h_low;
    p.p_stride = a.pitch;
    p.rows = s.rows;
    p.k = a.pitch;
    p.q = a.down;
    p.q_stride = a.pitch;
    p.row_mask = row_mask;
    p.out = static_cast<uint16_t*>(y);
    p.columns = s.out_features;
    p.partials = reinterpret_cast<float*>(ws + l.partials);
    const auto queue = static_cast<hipStream_t>(stream);
    hipError_t error = lsso_hip::launch_feed_forward_pack(l.plan.pack, s.dtype, queue);
    if (error == hipSuccess) {
        error = lsso_hip::launch_feed_forward_gate(a, queue);
    }
    if (error == hipSuccess) {
        error = lsso_hip::launch_feed_forward_product(p, queue);
    }
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "feed-forward launch");
}

int lsso_hip_feed_forward_backward_workspace_bytes(const lsso_hip_feed_forward_shape* shape, int64_t grad_stride,
                                                   int weights, size_t* bytes) {
    const int status = check_feed_forward(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (bytes == nullptr || grad_stride < shape->out_features) {
        return report(LSSO_HIP_EINVAL, "bytes must not be NULL and grad_stride at least out_features");
    }
    if (weights < 0 || weights > 7) {
        return report(LSSO_HIP_EINVAL, "weights must be 0 .. 7");
    }
    const bool wanted[3] = {(weights & 1) != 0, (weights & 2) != 0, (weights & 4) != 0};
    *bytes = backward_layout(*shape, grad_stride, wanted).plan.bytes;
    return LSSO_HIP_OK;
}

int lsso_hip_feed_forward_backward(const lsso_hip_feed_forward_shape* shape, const void* grad_y, int64_t grad_stride,
                                   const void* x, const void* gate_weight, const void* up_weight,
                                   const void* down_weight, const uint8_t* row_mask, const void* gates,
                                   const void* product, void* grad_x, void* grad_gate, void* grad_up, void* grad_down,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    const int status = check_feed_forward(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_feed_forward_shape& s = *shape;
    if (grad_stride < s.out_features) {
        return report(LSSO_HIP_EINVAL, "grad_stride must be at least out_features");
    }
    if (s.rows > 0 && (grad_y == nullptr || x == nullptr || gate_weight == nullptr || up_weight == nullptr ||
                       down_weight == nullptr || gates == nullptr || product == nullptr)) {
        return report(LSSO_HIP_EINVAL, "grad_y, x, the weights, gates and product must not be NULL");
    }
    if (!aligned(grad_y, 16) || !aligned(x, 16) || !aligned(gate_weight, 16) || !aligned(up_weight, 16) ||
        !aligned(down_weight, 16) || !aligned(gates, 16) || !aligned(product, 16)) {
        return report(LSSO_HIP_EINVAL, "grad_y, x, the weights, gates and product must be 16-byte aligned");
    }
    void* const outputs[3] = {grad_gate, grad_up, grad_down};
    const bool wanted[3] = {grad_gate != nullptr, grad_up != nullptr, grad_down != nullptr};
    FeedForwardLayout l = backward_layout(s, grad_stride, wanted);
    if (l.plan.bytes > 0 && (workspace == nullptr || workspace_bytes < l.plan.bytes || !aligned(workspace, 256))) {
        return report(LSSO_HIP_EINVAL,
                      "workspace must be 256-byte aligned and of lsso_hip_feed_forward_backward_workspace_bytes()");
    }
    char* ws = static_cast<char*>(workspace);
    const bool wide = s.weight_type == LSSO_HIP_F32;
    lsso_hip::FeedForwardArgs& a = l.plan.args;
    a.x = bind(&l.plan, l.x, x, s.rows, s.in_features, s.x_stride, false, ws);
    a.x_stride = l.x.stride;
    a.dy = bind(&l.plan, l.dy, grad_y, s.rows, s.out_features, grad_stride, false, ws);
    a.dy_stride = l.dy.stride;
    a.row_mask = row_mask;
    bind_gates(s, const_cast<void*>(gates), &a);
    a.grads = reinterpret_cast<uint16_t*>(ws + l.grads);
    uint16_t* const in_columns = reinterpret_cast<uint16_t*>(ws + l.in_columns);
    uint16_t* const down_columns = reinterpret_cast<uint16_t*>(ws + l.down_columns);
    a.down_columns = down_columns;
    const bool through = grad_x != nullptr || wanted[0] || wanted[1];   // dg and du are needed
    if (through) {
        transpose(&l.plan, down_weight, s.out_features, s.hidden, wide, down_columns, a.out_pitch);
    }
    if (grad_x != nullptr) {
        transpose(&l.plan, gate_weight, s.hidden, s.in_features, wide, in_columns, 2 * a.pitch);
        transpose(&l.plan, up_weight, s.hidden, s.in_features, wide, in_columns + a.pitch, 2 * a.pitch);
    }
    const auto queue = static_cast<hipStream_t>(stream);
    hipError_t error = hipSuccess;
    if (s.rows > 0) {
        error = lsso_hip::launch_feed_forward_pack(l.plan.pack, s.dtype, queue);
        if (error == hipSuccess && through) {
            error = lsso_hip::launch_feed_forward_grad(a, queue);
        }
    }
    if (error == hipSuccess && grad_x != nullptr && s.rows > 0) {
        lsso_hip::FeedForwardProduct& p = l.plan.product;
        p.type = s.dtype;
        p.p = a.grads;
        p.p_stride = 2 * a.pitch;
        p.rows = s.rows;
        p.k = 2 * a.pitch;
        p.q = in_columns;
        p.q_stride = 2 * a.pitch;
        p.row_mask = row_mask;
        p.out = static_cast<uint16_t*>(grad_x);
        p.columns = s.in_features;
        p.partials = reinterpret_cast<float*>(ws + l.partials);
        error = lsso_hip::launch_feed_forward_product(p, queue);
    }
    lsso_hip::FeedForwardWeights& w = l.plan.weights;
    if (error == hipSuccess && w.count > 0) {
        w.row_mask = row_mask;
        w.partials = reinterpret_cast<float*>(ws + l.weight_partials);
        lsso_hip::FeedForwardJoin join{};
        join.partials = w.partials;
        join.splits = s.rows > 0 ? w.splits : 0;
        join.split_floats = w.partial_floats;
        join.type = s.weight_type;
        int at = 0;
        for (int i = 0; i < 3; ++i) {
            if (!wanted[i]) {
                continue;
            }
            lsso_hip::WeightProduct& q = w.products[at];
            if (i < 2) {
                q.p = a.grads + i * a.pitch;
                q.q = a.x;
                q.q_stride = a.x_stride;
            } else {
                q.p = a.dy;
                q.p_stride = a.dy_stride;
                q.q = static_cast<const uint16_t*>(product);
            }
            join.outputs[at++] = {q.partial_offset, q.partial_pitch, q.out_rows, i < 2 ? s.in_features : s.hidden,
                                  outputs[i]};
        }
        if (s.rows > 0) {
            error = lsso_hip::launch_feed_forward_weights(w, queue);
        }
        if (error == hipSuccess) {
            error = lsso_hip::launch_feed_forward_join(join, at, queue);
        }
    }
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "feed-forward gradient launch");
}

int lsso_hip_embedding(const void* tokens, int token_bytes, int64_t count, const void* weight, int weight_type,
                       int64_t vocabulary, int64_t dim, int64_t weight_stride, float scale,
                       const uint8_t* row_mask, void* y, int y_type, void* stream) {
    const int status = check_embedding(tokens, token_bytes, count, vocabulary, dim);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (!value_type(weight_type) || !value_type(y_type)) {
        return report(LSSO_HIP_EINVAL, "weight and y must be float16, bfloat16 or float32");
    }
    if (weight_stride < dim) {
        return report(LSSO_HIP_EINVAL, "weight_stride must be at least dim");
    }
    if (count > 0 && (weight == nullptr || y == nullptr || !aligned(weight, type_bytes(weight_type)) ||
                      !aligned(y, type_bytes(y_type)))) {
        return report(LSSO_HIP_EINVAL, "weight and y must not be NULL and be aligned to their type");
    }
    lsso_hip::EmbeddingArgs args{};
    args.tokens = tokens;
    args.wide_tokens = token_bytes == 8;
    args.count = count;
    args.vocabulary = vocabulary;
    args.dim = dim;
    args.row_mask = row_mask;
    args.scale = scale;
    args.weight = weight;
    args.weight_stride = weight_stride;
    args.weight_type = weight_type;
    args.y = y;
    const hipError_t error = lsso_hip::launch_embedding(args, y_type, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "lookup_kernel launch");
}

int lsso_hip_embedding_grad_workspace_bytes(int64_t count, int64_t vocabulary, int64_t dim, size_t* bytes) {
    if (bytes == nullptr) {
        return report(LSSO_HIP_EINVAL, "bytes must not be NULL");
    }
    const int status = check_embedding(bytes, 4, count, vocabulary, dim);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    lsso_hip::EmbeddingArgs args{};
    args.count = count;
    args.vocabulary = vocabulary;
    args.dim = dim;
    lsso_hip::plan_embedding_grad(&args, bytes);
    return LSSO_HIP_OK;
}

int lsso_hip_embedding_grad(const void* tokens, int token_bytes, int64_t count, const void* grad_y, int grad_type,
                            int64_t grad_stride, int64_t vocabulary, int64_t dim, float scale,
                            const uint8_t* row_mask, int64_t padding_index, void* grad_weight, int weight_type,
                            void* workspace, size_t workspace_bytes, void* stream) {
    const int status = check_embedding(tokens, token_bytes, count, vocabulary, dim);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (!value_type(weight_type) || !value_type(grad_type)) {
        return report(LSSO_HIP_EINVAL, "grad_y and grad_weight must be float16, bfloat16 or float32");
    }
    if (count > 1 && grad_stride < dim) {
        return report(LSSO_HIP_EINVAL, "grad_stride must be at least dim");
    }
    if (padding_index < -1 || padding_index >= vocabulary) {
        return report(LSSO_HIP_EINVAL, "padding_index must be -1 or a row of the table");
    }
    if (grad_weight == nullptr || !aligned(grad_weight, type_bytes(weight_type)) ||
        (count > 0 && (grad_y == nullptr || !aligned(grad_y, type_bytes(grad_type))))) {
        return report(LSSO_HIP_EINVAL, "grad_y and grad_weight must not be NULL and be aligned to their type");
    }
    lsso_hip::EmbeddingArgs args{};
    args.tokens = tokens;
    args.wide_tokens = token_bytes == 8;
    args.count = count;
    args.vocabulary = vocabulary;
    args.dim = dim;
    args.row_mask = row_mask;
    args.scale = scale;
    args.weight_type = weight_type;
    args.grad_y = grad_y;
    args.grad_stride = grad_stride;
    args.padding_index = padding_index;
    args.grad_weight = grad_weight;
    size_t bytes = 0;
    lsso_hip::plan_embedding_grad(&args, &bytes);
    if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 256))) {
        return report(LSSO_HIP_EINVAL,
                      "workspace must be 256-byte aligned and of lsso_hip_embedding_grad_workspace_bytes()");
    }
    const hipError_t error =
        lsso_hip::launch_embedding_grad(args, workspace, grad_type, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "embedding gradient launch");
}

int lsso_hip_dropout_add(const void* x, const void* residual, int dtype, int64_t count, uint32_t threshold,
                         uint64_t seed, uint64_t offset, const int64_t* state, void* y, void* stream) {
    if (count < 0) {
        return report(LSSO_HIP_EINVAL, "count must not be negative");
    }
    if (count > (int64_t{1} << 34)) {
        return report(LSSO_HIP_EUNSUPPORTED, "dropout takes up to 2^34 elements");
    }
    if (!value_type(dtype)) {
        return report(LSSO_HIP_EINVAL, "dropout takes float16, bfloat16 or float32");
    }
    if (threshold > 65535) {
        return report(LSSO_HIP_EINVAL, "threshold must be 0 .. 65535");
    }
    if (count > 0 && (x == nullptr || y == nullptr)) {
        return report(LSSO_HIP_EINVAL, "x and y must not be NULL");
    }
    const uintptr_t bytes = type_bytes(dtype);
    if (!aligned(x, bytes) || !aligned(residual, bytes) || !aligned(y, bytes) || !aligned(state, 8)) {
        return report(LSSO_HIP_EINVAL, "x, residual, y and state must be aligned to their type");
    }
    lsso_hip::DropoutArgs args{};
    args.x = x;
    args.residual = residual;
    args.y = y;
    args.count = count;
    args.threshold = threshold;
    args.scale = 65536.0f / static_cast<float>(65536 - threshold);
    args.seed = seed;
    args.offset = offset;
    args.state = state;
    const hipError_t error = lsso_hip::launch_dropout(args, dtype, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "dropout_kernel launch");
}

}  // extern "C"
