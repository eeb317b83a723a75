// C ABI of the operators of the causal mixer (rotary positions, group norm,
// linear attention): host-side validation, workspace planning and
// stream-ordered launches, as in lsso_capi.hip.  No exception leaves these
// entries: nothing here allocates.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "lsso_hip.h"
#include "lsso_internal.h"

namespace {

using lsso_hip::report;
using lsso_hip::report_hip;

bool value_type(int type) { return type == LSSO_HIP_F16 || type == LSSO_HIP_BF16 || type == LSSO_HIP_F32; }
bool aligned(const void* pointer, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(pointer) % bytes == 0; }
uintptr_t type_bytes(int type) { return type == LSSO_HIP_F32 ? 4 : 2; }
size_t round256(size_t bytes) { return (bytes + 255) & ~static_cast<size_t>(255); }

constexpr int64_t kMostTokens = int64_t{1} << 40;   // of a tensor, and its strides: products stay within 63 bits
constexpr int64_t kMostHeads = 4096;
constexpr int64_t kMostRotary = 4096;
constexpr int64_t kMostChannels = 1 << 20;
constexpr int64_t kMostSamples = 1 << 30;
constexpr int64_t kMostLength = 1 << 30;
constexpr int64_t kMostBlocks = 1 << 22;            // two workgroups of 256 threads to each: fewer than 2^32 threads

bool strides_fit(int64_t batch, int64_t token, int64_t head) {
    return batch >= 0 && token >= 0 && head >= 0 && batch <= kMostTokens && token <= kMostTokens && head <= kMostTokens;
}

int check_group_norm(const lsso_hip_group_norm_shape* s) {
    if (s == nullptr) {
        return report(LSSO_HIP_EINVAL, "shape must not be NULL");
    }
    if (s->samples < 0 || s->length < 0 || s->channels <= 0 || s->groups <= 0 || s->channels % s->groups != 0) {
        return report(LSSO_HIP_EINVAL,
                      "samples and length must not be negative, groups must be positive and divide channels");
    }
    if (s->samples > kMostSamples || s->length > kMostLength || s->channels > kMostChannels ||
        (s->samples > 0 && s->length > (int64_t{1} << 40) / s->samples)) {
        return report(LSSO_HIP_EUNSUPPORTED,
                      "group norm takes up to 2^30 samples, 2^30 tokens in each, 2^40 in all and 2^20 channels");
    }
    if (!value_type(s->dtype)) {
        return report(LSSO_HIP_EUNSUPPORTED, "group norm takes float16, bfloat16 or float32");
    }
    if (s->parameter_type != s->dtype && s->parameter_type != LSSO_HIP_F32) {
        return report(LSSO_HIP_EUNSUPPORTED, "weight and bias must have x's type or float32");
    }
    if (s->activation != 0 && s->activation != LSSO_HIP_SILU && s->activation != LSSO_HIP_GELU) {
        return report(LSSO_HIP_EUNSUPPORTED, "activation must be 0, LSSO_HIP_SILU or LSSO_HIP_GELU");
    }
    if (!(s->eps >= 0.0f) || std::isinf(s->eps)) {
        return report(LSSO_HIP_EINVAL, "eps must be finite and not negative");
    }
    return LSSO_HIP_OK;
}

lsso_hip::GroupNormArgs group_norm_args(const lsso_hip_group_norm_shape& s) {
    lsso_hip::GroupNormArgs a{};
    a.samples = s.samples;
    a.length = s.length;
    a.channels = static_cast<int>(s.channels);
    a.groups = static_cast<int>(s.groups);
    a.parameter_type = s.parameter_type;
    a.activation = s.activation;
    a.eps = s.eps;
    return a;
}

struct GroupNormLayout {
    size_t kept = 0;        // floats
    size_t statistics = 0;  // offset of them in the workspace where they are not kept
    size_t sums = 0;
    size_t bytes = 0;
};

// Plans `a`; the workspace holds the partials first.
GroupNormLayout group_norm_layout(lsso_hip::GroupNormArgs* a, bool backward) {
    GroupNormLayout l;
    size_t partials = 0;
    lsso_hip::plan_group_norm(a, backward, &partials);
    l.bytes = round256(partials);
    if (a->team != 0) {
        return l;
    }
    l.kept = 2 * static_cast<size_t>(a->samples) * static_cast<size_t>(a->groups);
    if (backward) {
        l.sums = l.bytes;
    } else {
        l.statistics = l.bytes;
    }
    l.bytes += round256(sizeof(float) * l.kept);
    return l;
}

int check_linear_attention(const lsso_hip_linear_attention_shape* s) {
    if (s == nullptr) {
        return report(LSSO_HIP_EINVAL, "shape must not be NULL");
    }
    if (s->batch < 0 || s->length < 0 || s->heads <= 0 || s->kv_heads <= 0 || s->heads % s->kv_heads != 0 ||
        s->features <= 0 || s->value_features <= 0) {
        return report(LSSO_HIP_EINVAL,
                      "batch and length must not be negative, features must be positive, kv_heads must divide heads");
    }
    if (s->features > lsso_hip::kWalkFeatures || s->value_features > lsso_hip::kWalkFeatures) {
        return report(LSSO_HIP_EUNSUPPORTED, "linear attention takes up to 128 features and value features a head");
    }
    if (s->heads > kMostHeads || s->length > kMostLength || s->batch > kMostBlocks ||
        s->batch * s->heads > kMostBlocks) {
        return report(LSSO_HIP_EUNSUPPORTED,
                      "linear attention takes up to 2^30 tokens, 4,096 heads and 2^22 sequences times heads");
    }
    if (s->dtype != LSSO_HIP_F16 && s->dtype != LSSO_HIP_BF16) {
        return report(LSSO_HIP_EUNSUPPORTED, "linear attention takes float16 or bfloat16");
    }
    if (!std::isfinite(s->scale)) {
        return report(LSSO_HIP_EINVAL, "scale must be finite");
    }
    if (!strides_fit(s->q.batch, s->q.token, s->q.head) || !strides_fit(s->k.batch, s->k.token, s->k.head) ||
        !strides_fit(s->v.batch, s->v.token, s->v.head)) {
        return report(LSSO_HIP_EINVAL, "strides must not be negative");
    }
    return LSSO_HIP_OK;
}

lsso_hip::WalkTensor tensor(const void* data, const lsso_hip_head_strides& strides, int64_t heads_per) {
    return {data, strides.batch, strides.token, strides.head, static_cast<int>(heads_per)};
}

lsso_hip_head_strides dense(int64_t length, int64_t heads, int64_t features) {
    return {length * heads * features, heads * features, features};
}

// The same tensor from its last token to its first.
lsso_hip::WalkTensor turned(lsso_hip::WalkTensor t, int64_t length, int64_t bytes) {
    if (t.data != nullptr && length > 0) {
        t.data = static_cast<const char*>(t.data) + bytes * (length - 1) * t.token;
    }
    t.token = -t.token;
    return t;
}

// The forward's shape and the plan of every walk of it, made here alone: a workspace
// laid out for one plan must not be written under another.  (The backward's walks
// exchange features and value features; their states have as many values.)
lsso_hip::WalkArgs walk_args(const lsso_hip_linear_attention_shape& s, const float* log_decay, const uint8_t* mask) {
    lsso_hip::WalkArgs w{};
    w.batch = s.batch;
    w.length = s.length;
    w.heads = static_cast<int>(s.heads);
    w.features = static_cast<int>(s.features);
    w.out_features = static_cast<int>(s.value_features);
    w.log_decay = log_decay;
    w.mask = mask;
    w.mask_batch = s.length;
    w.mask_token = 1;
    lsso_hip::plan_walk(&w);
    return w;
}

struct AttentionLayout {
    size_t counts = 0;
    size_t states = 0;
    size_t partial = 0;       // FP32 gradients of every head, where heads share one
    size_t kept_floats = 0;   // of states
    size_t bytes = 0;
};

// The workspace of a walk: updates, counts and states (which a training forward
// keeps for its backward instead).
AttentionLayout attention_layout(const lsso_hip_linear_attention_shape& s, bool backward) {
    AttentionLayout l;
    const lsso_hip::WalkArgs w = walk_args(s, nullptr, nullptr);
    if (w.segments > 1) {
        const size_t state = static_cast<size_t>(s.batch * s.heads) * static_cast<size_t>(s.features * s.value_features);
        l.counts = round256(sizeof(float) * state * static_cast<size_t>(w.pieces));
        l.states = l.counts + round256(sizeof(int) * static_cast<size_t>(s.batch * w.pieces));
        l.kept_floats = state * static_cast<size_t>(w.segments);
        l.bytes = l.states + round256(sizeof(float) * l.kept_floats);
    }
    if (backward && s.kv_heads < s.heads) {
        const int64_t widest = s.features > s.value_features ? s.features : s.value_features;
        l.partial = l.bytes;
        l.bytes += round256(sizeof(float) * static_cast<size_t>(s.batch * s.length) *
                            static_cast<size_t>(s.heads * widest));
    }
    return l;
}

bool bad_workspace(const void* workspace, size_t given, size_t needed) {
    return needed > 0 && (workspace == nullptr || given < needed || !aligned(workspace, 256));
}

}  // namespace

extern "C" {

int lsso_hip_rotary(const lsso_hip_rotary_tensor* tensors, int count, int dtype, int64_t batch, int64_t length,
                    int64_t features, int64_t rotary_features, int layout, const double* frequencies, float amplitude,
                    int inverse, const void* position_ids, int position_type, int64_t position_batch_stride,
                    int64_t position_token_stride, void* stream) {
    if (tensors == nullptr || count < 1 || count > 2) {
        return report(LSSO_HIP_EINVAL, "rotary takes one or two tensors");
    }
    if (batch < 0 || length < 0 || features <= 0 || rotary_features < 2 || rotary_features % 2 != 0 ||
        rotary_features > features) {
        return report(LSSO_HIP_EINVAL,
                      "batch and length must not be negative, rotary_features must be even and in 2 .. features");
    }
    if (features > kMostRotary || batch > kMostTokens || length > kMostTokens ||
        (batch > 0 && length > kMostTokens / batch)) {
        return report(LSSO_HIP_EUNSUPPORTED, "rotary takes up to 4,096 features and 2^40 tokens");
    }
    if (!value_type(dtype)) {
        return report(LSSO_HIP_EUNSUPPORTED, "rotary takes float16, bfloat16 or float32");
    }
    if (layout != LSSO_HIP_ROTARY_INTERLEAVED && layout != LSSO_HIP_ROTARY_HALF) {
        return report(LSSO_HIP_EINVAL, "layout must be LSSO_HIP_ROTARY_INTERLEAVED or LSSO_HIP_ROTARY_HALF");
    }
    if (position_type < LSSO_HIP_IDS_NONE || position_type > LSSO_HIP_IDS_F64) {
        return report(LSSO_HIP_EINVAL, "position_type must be one of LSSO_HIP_IDS_*");
    }
    lsso_hip::RotaryArgs a{};
    const uintptr_t bytes = type_bytes(dtype);
    for (int i = 0; i < count; ++i) {
        const lsso_hip_rotary_tensor& t = tensors[i];
        if (t.heads <= 0 || !strides_fit(t.batch_stride, t.token_stride, t.head_stride)) {
            return report(LSSO_HIP_EINVAL, "heads must be positive and strides not negative");
        }
        if (t.heads > kMostHeads) {
            return report(LSSO_HIP_EUNSUPPORTED, "rotary takes up to 4,096 heads");
        }
        if (batch * length > 0 && (t.x == nullptr || t.y == nullptr || !aligned(t.x, bytes) || !aligned(t.y, bytes))) {
            return report(LSSO_HIP_EINVAL, "x and y must not be NULL and be aligned to their type");
        }
        a.tensors[i] = {t.x, t.y, t.batch_stride, t.token_stride, t.head_stride, static_cast<int>(t.heads)};
    }
    if (batch * length == 0) {
        return LSSO_HIP_OK;
    }
    if (frequencies == nullptr || !aligned(frequencies, 8)) {
        return report(LSSO_HIP_EINVAL, "frequencies must not be NULL and be aligned to float64");
    }
    const uintptr_t id_bytes = position_type == LSSO_HIP_IDS_I64 || position_type == LSSO_HIP_IDS_F64 ? 8 : 4;
    if (position_type != LSSO_HIP_IDS_NONE && (position_ids == nullptr || !aligned(position_ids, id_bytes))) {
        return report(LSSO_HIP_EINVAL, "position_ids must not be NULL and be aligned to their type");
    }
    a.count = count;
    a.batch = batch;
    a.length = length;
    a.features = static_cast<int>(features);
    a.half = static_cast<int>(rotary_features / 2);
    a.frequencies = frequencies;
    a.amplitude = amplitude;
    a.sign = inverse != 0 ? -1.0f : 1.0f;
    a.positions = position_ids;
    a.position_type = position_type;
    a.position_batch_stride = position_batch_stride;
    a.position_token_stride = position_token_stride;
    const hipError_t error = lsso_hip::launch_rotary(a, dtype, layout, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "rotary_kernel launch");
}

int lsso_hip_group_norm_sizes(const lsso_hip_group_norm_shape* shape, size_t* kept_floats, size_t* forward_bytes,
                              size_t* backward_bytes) {
    const int status = check_group_norm(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (kept_floats == nullptr || forward_bytes == nullptr || backward_bytes == nullptr) {
        return report(LSSO_HIP_EINVAL, "kept_floats and the bytes must not be NULL");
    }
    lsso_hip::GroupNormArgs a = group_norm_args(*shape);
    const GroupNormLayout l = group_norm_layout(&a, false);
    *kept_floats = l.kept;
    *forward_bytes = l.bytes;
    *backward_bytes = group_norm_layout(&a, true).bytes;
    return LSSO_HIP_OK;
}

int lsso_hip_group_norm(const lsso_hip_group_norm_shape* shape, const void* x, const void* weight, const void* bias,
                        const uint8_t* row_mask, float* statistics, void* y, void* workspace, size_t workspace_bytes,
                        void* stream) {
    const int status = check_group_norm(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_group_norm_shape& s = *shape;
    if (s.samples * s.length == 0) {
        return LSSO_HIP_OK;
    }
    const uintptr_t bytes = type_bytes(s.dtype);
    const uintptr_t parameter_bytes = type_bytes(s.parameter_type);
    if (x == nullptr || y == nullptr || !aligned(x, bytes) || !aligned(y, bytes)) {
        return report(LSSO_HIP_EINVAL, "x and y must not be NULL and be aligned to their type");
    }
    if (!aligned(weight, parameter_bytes) || !aligned(bias, parameter_bytes) || !aligned(statistics, 4)) {
        return report(LSSO_HIP_EINVAL, "weight, bias and statistics must be aligned to their type");
    }
    lsso_hip::GroupNormArgs a = group_norm_args(s);
    const GroupNormLayout l = group_norm_layout(&a, false);
    if (bad_workspace(workspace, workspace_bytes, l.bytes)) {
        return report(LSSO_HIP_EINVAL, "workspace must be 256-byte aligned and of lsso_hip_group_norm_sizes()");
    }
    char* ws = static_cast<char*>(workspace);
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.row_mask = row_mask;
    a.y = y;
    a.partials = reinterpret_cast<float*>(ws);
    a.statistics = statistics != nullptr || l.kept == 0 ? statistics : reinterpret_cast<float*>(ws + l.statistics);
    const hipError_t error = lsso_hip::launch_group_norm(a, s.dtype, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "group norm launch");
}

int lsso_hip_group_norm_backward(const lsso_hip_group_norm_shape* shape, const void* grad_y, const void* x,
                                 const void* weight, const void* bias, const uint8_t* row_mask,
                                 const float* statistics, void* grad_x, void* grad_weight, void* grad_bias,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const int status = check_group_norm(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_group_norm_shape& s = *shape;
    const bool rows = s.samples * s.length > 0;
    const uintptr_t bytes = type_bytes(s.dtype);
    const uintptr_t parameter_bytes = type_bytes(s.parameter_type);
    if (rows && (x == nullptr || grad_y == nullptr || !aligned(x, bytes) || !aligned(grad_y, bytes) ||
                 !aligned(grad_x, bytes))) {
        return report(LSSO_HIP_EINVAL, "x, grad_y and grad_x must be aligned to their type and given");
    }
    if (!aligned(weight, parameter_bytes) || !aligned(bias, parameter_bytes) ||
        !aligned(grad_weight, parameter_bytes) || !aligned(grad_bias, parameter_bytes)) {
        return report(LSSO_HIP_EINVAL, "weight, bias and their gradients must be aligned to their type");
    }
    lsso_hip::GroupNormArgs a = group_norm_args(s);
    const GroupNormLayout l = group_norm_layout(&a, true);
    if (rows && l.kept > 0 && (statistics == nullptr || !aligned(statistics, 4))) {
        return report(LSSO_HIP_EINVAL, "statistics must be those that the forward kept");
    }
    if (bad_workspace(workspace, workspace_bytes, l.bytes)) {
        return report(LSSO_HIP_EINVAL, "workspace must be 256-byte aligned and of lsso_hip_group_norm_sizes()");
    }
    char* ws = static_cast<char*>(workspace);
    a.x = x;
    a.dy = grad_y;
    a.weight = weight;
    a.bias = bias;
    a.row_mask = row_mask;
    a.statistics = const_cast<float*>(statistics);
    a.dx = grad_x;
    a.grad_weight = grad_weight;
    a.grad_bias = grad_bias;
    a.partials = reinterpret_cast<float*>(ws);
    a.sums = reinterpret_cast<float*>(ws + l.sums);
    const hipError_t error = lsso_hip::launch_group_norm_backward(a, s.dtype, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "group norm gradient launch");
}

int lsso_hip_linear_attention_sizes(const lsso_hip_linear_attention_shape* shape, size_t* kept_floats,
                                    size_t* forward_bytes, size_t* backward_bytes) {
    const int status = check_linear_attention(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    if (kept_floats == nullptr || forward_bytes == nullptr || backward_bytes == nullptr) {
        return report(LSSO_HIP_EINVAL, "kept_floats and the bytes must not be NULL");
    }
    const AttentionLayout l = attention_layout(*shape, false);
    *kept_floats = l.kept_floats;
    *forward_bytes = l.bytes;
    *backward_bytes = attention_layout(*shape, true).bytes;
    return LSSO_HIP_OK;
}

int lsso_hip_linear_attention(const lsso_hip_linear_attention_shape* shape, const void* q, const void* k,
                              const void* v, const float* log_decay, const uint8_t* row_mask,
                              const float* initial_state, float* kept, void* y, float* final_state, void* workspace,
                              size_t workspace_bytes, void* stream) {
    const int status = check_linear_attention(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_linear_attention_shape& s = *shape;
    if (s.batch == 0 || (s.length == 0 && final_state == nullptr)) {
        return LSSO_HIP_OK;
    }
    if (s.length > 0 && (q == nullptr || k == nullptr || v == nullptr || y == nullptr || !aligned(q, 2) ||
                         !aligned(k, 2) || !aligned(v, 2) || !aligned(y, 2))) {
        return report(LSSO_HIP_EINVAL, "q, k, v and y must not be NULL and be aligned to their type");
    }
    if (log_decay == nullptr || !aligned(log_decay, 4) || !aligned(initial_state, 4) || !aligned(final_state, 4) ||
        !aligned(kept, 4)) {
        return report(LSSO_HIP_EINVAL, "log_decay must not be NULL, it and the states be aligned to float32");
    }
    const AttentionLayout l = attention_layout(s, false);
    if (bad_workspace(workspace, workspace_bytes, l.bytes)) {
        return report(LSSO_HIP_EINVAL,
                      "workspace must be 256-byte aligned and of lsso_hip_linear_attention_sizes()");
    }
    char* ws = static_cast<char*>(workspace);
    lsso_hip::WalkArgs w = walk_args(s, log_decay, row_mask);
    w.a = tensor(q, s.q, 1);
    w.b = tensor(k, s.k, s.heads / s.kv_heads);
    w.c = tensor(v, s.v, s.heads / s.kv_heads);
    w.out = tensor(y, dense(s.length, s.heads, s.value_features), 1);
    w.scale_within = s.scale;
    w.scale_across = s.scale;
    w.scale_update = 1.0f;
    w.first = initial_state;
    w.first_row = s.value_features;
    w.first_column = 1;
    w.last = final_state;
    w.updates = reinterpret_cast<float*>(ws);
    w.counts = reinterpret_cast<int*>(ws + l.counts);
    w.states = kept != nullptr ? kept : reinterpret_cast<float*>(ws + l.states);
    w.states_row = s.value_features;
    w.states_column = 1;
    const hipError_t error = lsso_hip::launch_walk(w, s.dtype, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "linear attention launch");
}

int lsso_hip_linear_attention_backward(const lsso_hip_linear_attention_shape* shape, const void* grad_y,
                                       const lsso_hip_head_strides* grad_strides, const float* grad_final_state,
                                       const void* q, const void* k, const void* v, const float* log_decay,
                                       const uint8_t* row_mask, const float* initial_state, const float* kept,
                                       void* grad_q, void* grad_k, void* grad_v, float* grad_initial_state,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    const int status = check_linear_attention(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_linear_attention_shape& s = *shape;
    if (grad_strides == nullptr || !strides_fit(grad_strides->batch, grad_strides->token, grad_strides->head)) {
        return report(LSSO_HIP_EINVAL, "grad_strides must not be NULL or negative");
    }
    if (s.batch == 0 || (s.length == 0 && grad_initial_state == nullptr)) {
        return LSSO_HIP_OK;
    }
    if (s.length > 0 && (q == nullptr || k == nullptr || v == nullptr || grad_y == nullptr || !aligned(q, 2) ||
                         !aligned(k, 2) || !aligned(v, 2) || !aligned(grad_y, 2))) {
        return report(LSSO_HIP_EINVAL, "q, k, v and grad_y must not be NULL and be aligned to their type");
    }
    if (log_decay == nullptr || !aligned(log_decay, 4) || !aligned(initial_state, 4) || !aligned(grad_final_state, 4) ||
        !aligned(grad_initial_state, 4) || !aligned(kept, 4) || !aligned(grad_q, 2) || !aligned(grad_k, 2) ||
        !aligned(grad_v, 2)) {
        return report(LSSO_HIP_EINVAL, "log_decay must not be NULL, it, the states and the gradients be aligned");
    }
    const AttentionLayout l = attention_layout(s, true);
    if (bad_workspace(workspace, workspace_bytes, l.bytes)) {
        return report(LSSO_HIP_EINVAL,
                      "workspace must be 256-byte aligned and of lsso_hip_linear_attention_sizes()");
    }
    char* ws = static_cast<char*>(workspace);
    const auto queue = static_cast<hipStream_t>(stream);
    const int64_t shared = s.heads / s.kv_heads;
    const lsso_hip::WalkTensor tq = tensor(q, s.q, 1);
    const lsso_hip::WalkTensor tk = tensor(k, s.k, shared);
    const lsso_hip::WalkTensor tv = tensor(v, s.v, shared);
    const lsso_hip::WalkTensor tdy = tensor(grad_y, *grad_strides, 1);
    const auto planned = [&](const lsso_hip::WalkTensor& a, const lsso_hip::WalkTensor& b,
                             const lsso_hip::WalkTensor& c, int64_t features, int64_t out_features) {
        lsso_hip::WalkArgs w = walk_args(s, log_decay, row_mask);
        w.a = a;
        w.b = b;
        w.c = c;
        w.features = static_cast<int>(features);
        w.out_features = static_cast<int>(out_features);
        w.scale_within = s.scale;
        w.updates = reinterpret_cast<float*>(ws);
        w.counts = reinterpret_cast<int*>(ws + l.counts);
        w.states = reinterpret_cast<float*>(ws + l.states);
        w.states_row = out_features;
        w.states_column = 1;
        return w;
    };
    hipError_t error = hipSuccess;
    if (grad_q != nullptr && s.length > 0) {
        lsso_hip::WalkArgs w = planned(tdy, tv, tk, s.value_features, s.features);
        w.out = tensor(grad_q, dense(s.length, s.heads, s.features), 1);
        w.scale_across = s.scale;
        w.scale_update = 1.0f;
        w.first = initial_state;   // S transposed
        w.first_row = 1;
        w.first_column = s.value_features;
        if (kept != nullptr) {   // the forward's, read transposed
            w.reuse = 1;
            w.states = const_cast<float*>(kept);
            w.states_row = 1;
            w.states_column = s.value_features;
        }
        error = lsso_hip::launch_walk(w, s.dtype, queue);
    }
    // To the front: S's gradient, from that of the last state on.  dk's states are
    // dv's, transposed.
    bool walked = false;
    const auto back = [&](const lsso_hip::WalkTensor& a, const lsso_hip::WalkTensor& b, const lsso_hip::WalkTensor& c,
                          int64_t features, int64_t out_features, void* grad, bool transposed, float* first_state) {
        const bool summed = shared > 1 && grad != nullptr;
        lsso_hip::WalkArgs w = planned(turned(a, s.length, 2), turned(b, s.length, 2), turned(c, s.length, 2),
                                       features, out_features);
        if (row_mask != nullptr && s.length > 0) {
            w.mask = row_mask + (s.length - 1);
            w.mask_token = -1;
        }
        void* to = summed ? static_cast<void*>(ws + l.partial) : grad;
        w.wide_out = summed ? 1 : 0;
        w.out = turned(tensor(to, dense(s.length, s.heads, out_features), 1), s.length, summed ? 4 : 2);
        w.scale_across = 1.0f;
        w.scale_update = s.scale;
        w.shift = 1;
        w.first = grad_final_state;
        w.first_row = transposed ? 1 : out_features;
        w.first_column = transposed ? features : 1;
        w.last = first_state;
        if (walked) {
            w.reuse = 1;
            w.states_row = 1;
            w.states_column = features;
        }
        walked = true;
        error = lsso_hip::launch_walk(w, s.dtype, queue);
        if (error == hipSuccess && summed && s.length > 0) {
            lsso_hip::HeadSumArgs sum{};
            sum.partial = reinterpret_cast<const float*>(ws + l.partial);
            sum.out = grad;
            sum.rows = s.batch * s.length;
            sum.kv_heads = static_cast<int>(s.kv_heads);
            sum.shared = static_cast<int>(shared);
            sum.features = static_cast<int>(out_features);
            error = lsso_hip::launch_head_sum(sum, s.dtype, queue);
        }
    };
    if (error == hipSuccess && ((grad_v != nullptr && s.length > 0) || grad_initial_state != nullptr)) {
        back(tk, tq, tdy, s.features, s.value_features, grad_v, false, grad_initial_state);
    }
    if (error == hipSuccess && grad_k != nullptr && s.length > 0) {
        back(tv, tdy, tq, s.value_features, s.features, grad_k, true, nullptr);
    }
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "linear attention gradient launch");
}

int lsso_hip_linear_attention_step(const lsso_hip_linear_attention_shape* shape, const void* q, const void* k,
                                   const void* v, const float* log_decay, const uint8_t* row_mask, float* state,
                                   int64_t state_batch_stride, void* y, void* stream) {
    const int status = check_linear_attention(shape);
    if (status != LSSO_HIP_OK) {
        return status;
    }
    const lsso_hip_linear_attention_shape& s = *shape;
    if (s.length != 1) {
        return report(LSSO_HIP_EINVAL, "a step takes one token of each sequence");
    }
    if (s.batch > 1 && (state_batch_stride < s.heads * s.features * s.value_features ||
                        state_batch_stride > kMostTokens)) {
        return report(LSSO_HIP_EINVAL, "the states must not overlap");
    }
    if (s.batch == 0) {
        return LSSO_HIP_OK;
    }
    if (q == nullptr || k == nullptr || v == nullptr || y == nullptr || !aligned(q, 2) || !aligned(k, 2) ||
        !aligned(v, 2) || !aligned(y, 2)) {
        return report(LSSO_HIP_EINVAL, "q, k, v and y must not be NULL and be aligned to their type");
    }
    if (log_decay == nullptr || state == nullptr || !aligned(log_decay, 4) || !aligned(state, 4)) {
        return report(LSSO_HIP_EINVAL, "log_decay and state must not be NULL and be aligned to float32");
    }
    lsso_hip::AttentionStepArgs a{};
    const int64_t shared = s.heads / s.kv_heads;
    a.q = tensor(q, s.q, 1);
    a.k = tensor(k, s.k, shared);
    a.v = tensor(v, s.v, shared);
    a.y = y;
    a.batch = s.batch;
    a.heads = static_cast<int>(s.heads);
    a.features = static_cast<int>(s.features);
    a.value_features = static_cast<int>(s.value_features);
    a.log_decay = log_decay;
    a.mask = row_mask;
    a.scale = s.scale;
    a.state = state;
    a.state_batch = state_batch_stride;
    const hipError_t error = lsso_hip::launch_attention_step(a, s.dtype, static_cast<hipStream_t>(stream));
    return error == hipSuccess ? LSSO_HIP_OK : report_hip(error, "attention_step_kernel launch");
}

}  // extern "C"
