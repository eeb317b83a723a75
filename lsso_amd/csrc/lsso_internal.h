// Kernel argument blocks and launchers shared between the kernel translation
// units and the C ABI.
#pragma once

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace lsso_hip {

// Events recorded by kernel dispatches themselves (hipExtLaunchKernel):
// `start` with the begin of the next dispatch, `stop` with the end of every
// dispatch, so that after a group of launches it holds the last one's end.
// Set per stage by the timed entry point around its own launches and cleared
// before it returns; unset, dispatches are plain launches.  Unlike
// hipEventRecord, this adds no queue packet between the kernels.
struct DispatchEvents {
    hipEvent_t start = nullptr;
    hipEvent_t stop = nullptr;
};
DispatchEvents& dispatch_events();   // this thread's

template <typename... KArgs, typename... Args>
inline void dispatch(void (*kernel)(KArgs...), dim3 grid, dim3 block, hipStream_t stream, Args... args) {
    DispatchEvents& events = dispatch_events();
    if (events.start == nullptr && events.stop == nullptr) {
        hipLaunchKernelGGL(kernel, grid, block, 0, stream, args...);
        return;
    }
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, events.start, events.stop, 0, args...);
    events.start = nullptr;
}

constexpr int kMaxPairs = 32;

struct PhaseArgs {
    const float* positions;  // centered positions or nullptr (default grid)
    uint32_t* phases;        // packed FP16 (cos, sin), [count]
    int64_t count;           // (batches) * length * pairs
    int64_t length;
    int pairs;
    float inverse_frequency[kMaxPairs];
};

// Centred positions and valid counts from a mask and position ids.
struct GeometryArgs {
    const uint8_t* mask;        // [rows, length] or nullptr
    const void* positions;      // ids, or nullptr (0 .. length - 1)
    int64_t position_batch_stride;
    int64_t position_token_stride;
    int64_t rows;               // samples, or 1 (one grid shared by all samples)
    int64_t length;
    float* centered;            // [rows, length]
    float* counts;              // [rows] (written when mask is set)
};

struct ReduceArgs {
    const uint16_t* projected;  // BF16 [B, N, width] (relation columns)
    const uint16_t* content;    // BF16 rows whose head-h columns are contracted with A
    int64_t content_stride;     // elements between consecutive tokens of `content`
    int gram;                   // also accumulate G = A^T A
    const uint32_t* phases;
    float* partials;            // [B, H, chunks, partial_stride]
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    int64_t width;              // heads * rank + heads * head_dim
    int64_t phase_batch_stride; // 0 (shared) or length * pairs
    int64_t chunks;
    int64_t chunk_tokens;       // multiple of 32
    int64_t column_groups;
    int64_t partial_stride;     // rank * rank + rank * head_dim
    int64_t total_waves;
    int64_t group_heads;        // staged form: heads per workgroup (0: one wave per work item)
};

struct SolveArgs {
    const float* partials;
    int64_t chunks;
    int64_t partial_stride;
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    const float* base;          // [H, R, R]
    const float* drive;         // [H, d, R]
    const float* eta_raw;       // [H]
    const float* valid_counts;  // [B] or nullptr
    float* zbuf;                // [B*H, R, d]
    uint16_t* mop;              // apply operand records
    float* tape;                // optional
    int64_t tape_stride;
};

struct ApplyArgs {
    const uint16_t* projected;
    const uint32_t* phases;
    const uint16_t* mop;
    const float* eta_raw;
    uint16_t* output;           // BF16 [B, N, H*d]
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    int64_t width;
    int64_t out_width;
    int64_t phase_batch_stride;
    int64_t chunks;
    int64_t chunk_tokens;       // multiple of 16
    int64_t feature_blocks;     // ceil(head_dim / 16)
    int64_t block_groups;       // ceil(feature_blocks / NFBW)
    int64_t total_waves;
    int64_t group_heads;        // staged form: heads per workgroup (0: one wave per work item)
    int64_t ranges;             // staged form: token ranges per sample
    int64_t range_tokens;       // staged form: tokens per range (a multiple of 16)
};

// Apply fused with the output projection: y = cast(bf16(mixed) bf16(W_o)^T
// + b_o) with mixed = eta C + rot(R) M' computed per 64-token tile in LDS.
struct MixProjectArgs {
    const uint16_t* projected;  // BF16 [B, N, width]
    const uint32_t* phases;
    const uint16_t* mop;        // apply operand records
    const float* eta_raw;       // [H]
    const float* weight;        // FP32 [D, D] (D = H * head_dim)
    const float* bias;          // FP32 [D] or nullptr
    const uint8_t* row_mask;    // [B * N] or nullptr
    void* y;                    // FP16/BF16 [B, N, D]
    uint16_t* mixed;            // BF16 [B, N, D] (the apply output, kept for training) or nullptr
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    int64_t width;
    int64_t out_features;       // D
    int64_t feature_blocks;     // head_dim / 16
    int64_t phase_batch_stride;
    int64_t ranges;             // token ranges per sample (one workgroup each)
    int64_t range_tokens;       // multiple of the 64-token tile
};

// Backward of the mixer (one compact system per workgroup).
struct BwdSolveArgs {
    const float* partials;      // S-part holds A^T dY per chunk
    int64_t chunks;
    int64_t partial_stride;
    const float* tape;          // [L | Theta | (I+K)^-1 | L^-1 | Z | U] per system
    int64_t tape_stride;
    const float* drive;         // [H, d, R]
    const float* eta_raw;       // [H]
    const float* valid_counts;  // [B] or nullptr
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    uint16_t* records;          // token-map operand records per system
    int64_t record_stride;      // in bf16
    int64_t off_m, off_e, off_g, off_f;
    int feature_k32;
    float* dtheta_part;         // [B*H, R, R]
    float* ddrive_part;         // [B*H, d, R]
    float* deta_part;           // [B*H]
};

struct BwdApplyArgs {
    const uint16_t* projected;  // BF16 [B, N, width]
    const uint16_t* grad_output;// BF16 [B, N, H*d]
    int64_t grad_stride;        // H*d
    const uint32_t* phases;
    int64_t phase_batch_stride;
    const uint16_t* records;
    int64_t record_stride;
    int64_t off_m, off_e, off_g, off_f;
    const float* eta_raw;
    uint16_t* grad_projected;   // BF16 [B, N, width]
    float* dot_part;            // [B*H, chunks]: <dY, C> per chunk
    float* column_part;         // [B*chunks, width]: column sums of grad_projected, or nullptr
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    int64_t width;
    int64_t chunks;
    int64_t chunk_tokens;       // multiple of 16
    int64_t total_waves;
};

struct ParamReduceArgs {
    const float* dtheta_part;
    const float* ddrive_part;
    const float* deta_part;
    const float* dot_part;
    const float* eta_raw;
    float* grad_base;           // [H, R, R]
    float* grad_drive;          // [H, d, R]
    float* grad_eta;            // [H]
    int64_t batch;
    int64_t heads;
    int64_t rank;
    int64_t head_dim;
    int64_t chunks;
};

struct LinearArgs {
    const void* x;
    int64_t rows;
    int64_t in_features;
    int64_t x_stride;
    const float* weight;        // FP32 [out, in]
    const float* bias;          // FP32 [out] or nullptr
    const uint8_t* row_mask;    // [rows] or nullptr; 0 rows are zeroed
    int64_t out_features;
    void* y;
    int64_t tiles;              // ceil(rows / tile_rows)
    int64_t column_groups;
    int vector;                 // x and y rows are whole aligned 16-byte pieces
};

// Upstream-gradient pass of the projection's backward: BF16 copy and FP32
// column sums of g [rows, cols] in one read.
struct GradColumnsArgs {
    const void* g;              // FP16/BF16 [rows, cols], row stride g_stride
    int64_t rows;
    int64_t cols;
    int64_t g_stride;
    const uint8_t* row_mask;    // [rows] or nullptr; 0 rows count as zero
    uint16_t* g_bf16;           // BF16 [rows, cols] contiguous, or nullptr
    float* partials;            // [splits, cols] column sums per split, or nullptr
    int64_t rows_per_split;
    int chunks_per_slab;        // 8-column chunks per workgroup: divides 256
};

// Input projection fused with the L-reductions (one pass over x per head
// group): packed = bf16(x W^T + b) per 64-token tile in LDS, contracted into
// the G / S partials of each head of the group and optionally written out.
struct ProjectReduceArgs {
    const void* x;              // FP16/BF16 [B, N, D], rows contiguous
    const float* weight;        // FP32 [width, D]
    const float* bias;          // FP32 [width] or nullptr
    const uint8_t* row_mask;    // [B * N] or nullptr; 0 rows project to zero
    const uint32_t* phases;
    int64_t phase_batch_stride;
    uint16_t* packed;           // BF16 [B, N, width] or nullptr
    float* partials;            // [B, H, chunks, partial_stride]
    int64_t batch;
    int64_t length;
    int64_t heads;
    int64_t head_dim;
    int64_t in_features;        // D
    int64_t width;              // H * (rank + head_dim)
    int64_t chunks;
    int64_t chunk_tokens;       // multiple of the 64-token tile
    int64_t partial_stride;
    int64_t group_heads;        // heads per head group
    int64_t head_groups;
};

// Weight and bias gradient of the biased projection: FP32 partials per row
// split of sum_m bf16(g[m][n]) bf16(x[m][k]) and of sum_m g[m][n].
struct WeightGradArgs {
    const void* g;              // FP16/BF16 [rows, out_features], row stride g_stride
    int64_t g_stride;
    const void* x;              // FP16/BF16 [rows, in_features], row stride x_stride
    int64_t x_stride;
    const uint8_t* row_mask;    // [rows] or nullptr; 0 rows count as zero
    int64_t rows;
    int64_t out_features;
    int64_t in_features;
    float* partials;            // [splits, out_features, in_features]
    float* bias_partials;       // [splits, out_features] or nullptr
    int64_t rows_per_split;     // multiple of 32
    int64_t splits;
    int64_t tiles_n;            // output tiles (set by the launcher)
    int64_t tiles_k;
    int vec;                    // 16-byte loads of g and x are legal
    int dealt;                  // row splits are dealt to the XCDs (set by the launcher)
    int large;                  // 256 x 256 output tiles, else 128 x 128 (set by the launcher)
};

// Residual dropout (lsso_dropout.hip).
struct DropoutArgs {
    const void* x;
    const void* residual;       // or nullptr
    void* y;
    int64_t count;
    uint32_t threshold;         // drop probability in units of 2^-16
    float scale;                // 65536 / (65536 - threshold)
    uint64_t seed;
    uint64_t offset;
    const int64_t* state;       // device (seed, offset): replaces seed, adds to offset; or nullptr
};

// Token embedding and its gradient (lsso_embedding.hip).
struct EmbeddingArgs {
    const void* tokens;         // int32 or int64 [count]
    int wide_tokens;            // int64
    int64_t count;
    int64_t vocabulary;
    int64_t dim;
    const uint8_t* row_mask;    // [count] or nullptr; 0 rows are zeros and count nowhere
    float scale;
    // Lookup.
    const void* weight;         // [vocabulary, dim], row stride weight_stride
    int64_t weight_stride;
    int weight_type;            // also of grad_weight
    void* y;                    // [count, dim]
    int64_t block_rows;
    // Gradient.
    const void* grad_y;         // [count, dim], row stride grad_stride
    int64_t grad_stride;
    int64_t padding_index;      // or -1
    void* grad_weight;          // [vocabulary, dim]
    uint32_t* histograms;       // [tiles, digits of the pass]
    int64_t tile_tokens;
    int64_t tiles;
    int key_bits;
    int passes;
    const uint32_t* keys;       // sorted ids, then `vocabulary` for what counts nowhere
    const uint32_t* index;      // token of each sorted position
    float* partials;            // [chunks, 2, dim]
    int64_t chunk_tokens;
    int64_t chunks;
    size_t off_sorted[4];
    size_t off_histograms;
    size_t off_partials;
};

// One pass of the gradient's radix sort; without inputs the tokens themselves.
struct SortPass {
    const uint32_t* keys_in;
    const uint32_t* index_in;
    uint32_t* keys_out;
    uint32_t* index_out;
    int shift;
    int bits;
    int part;    // of the gradient that the first of the pass' two launches clears
    int parts;
};

// Gated feed-forward block (lsso_feed_forward.hip).  All matrices are 16-bit of
// `type` unless they say otherwise; pitches are multiples of 8.
constexpr int kFewRows = 32;   // up to here without tiles

struct FeedForwardArgs {
    int type;
    int activation;
    int64_t rows;
    int64_t hidden;
    int64_t out_features;
    int64_t in_pitch;           // columns of x, gate and up, zeros past in_features
    int64_t pitch;              // columns of h: hidden rounded up
    int64_t out_pitch;          // columns of dy
    const uint16_t* x;          // [rows, in_pitch], row stride x_stride
    int64_t x_stride;
    const uint16_t* gate;       // [hidden, in_pitch]
    const uint16_t* up;         // [hidden, in_pitch]
    const uint16_t* down;       // [out_features, pitch]
    const uint16_t* down_columns;   // its transpose [hidden, out_pitch], of the backward
    const uint8_t* row_mask;    // [rows] or nullptr
    uint16_t* h;                // [rows, pitch]
    uint16_t* h_low;            // what rounding h left, of up to kFewRows rows
    uint16_t* gates;            // [rows, 2, pitch]: u act'(g), act(g), or their upper 16 bits; or nullptr
    char* gates_lower;          // [rows, lower_pitch]: the other bits of fine factors; or nullptr
    int64_t lower_pitch;
    const uint16_t* dy;         // [rows, out_pitch], row stride dy_stride
    int64_t dy_stride;
    uint16_t* grads;            // [rows, 2, pitch]: dg, du
    int stages;                 // set by the launcher, as the tiles
    int q_tiles;
    int tiles;
};

struct FeedForwardProduct {
    int type;
    const uint16_t* p;          // [rows, k], row stride p_stride
    const uint16_t* p_low;      // a second part of p, added to it, of up to kFewRows rows; or nullptr
    int64_t p_stride;
    int64_t rows;
    int64_t k;                  // a multiple of 8
    const uint16_t* q;          // [columns, k], row stride q_stride
    int64_t q_stride;
    const uint8_t* row_mask;
    uint16_t* out;              // [rows, columns] contiguous
    int64_t columns;
    float* partials;            // [splits, rows, partial_pitch], unused with one split
    int64_t partial_pitch;
    int stages;                 // set by plan_product, as what follows
    int split_stages;
    int splits;
    int q_tiles;                // set by the launcher
    int tiles;
};

struct WeightProduct {
    const uint16_t* p;          // [rows, p_columns], row stride p_stride
    int64_t p_stride;
    int64_t p_columns;
    const uint16_t* q;          // [rows, q_columns], row stride q_stride
    int64_t q_stride;
    int64_t q_columns;
    int64_t out_rows;
    int64_t partial_pitch;      // columns of the product, a multiple of 8
    int64_t partial_offset;     // set by plan_weights, as the tiles
    int64_t q_tiles;
    int64_t tiles;
};
constexpr int kWeightSplitRows = 32768;   // most rows of a split

struct FeedForwardWeights {
    int type;
    int count;
    WeightProduct products[3];
    int64_t rows;
    const uint8_t* row_mask;
    float* partials;            // [splits, partial_floats]
    int64_t partial_floats;
    int64_t split_rows;
    int64_t splits;
    int64_t tiles;              // of one split
    int large;                  // 256 x 256 tiles, else 128 x 128
};

struct JoinOutput {
    int64_t offset;
    int64_t pitch;
    int64_t rows;
    int64_t columns;
    void* out;                  // [rows, columns] contiguous
};

struct FeedForwardJoin {
    const float* partials;
    int64_t splits;
    int64_t split_floats;
    const uint8_t* row_mask;    // of the outputs' rows, or nullptr
    int type;                   // of the outputs
    JoinOutput outputs[3];
};

struct PackMatrix {
    const void* from;           // [rows, columns], row stride `stride`
    int64_t stride;
    int64_t rows;
    int64_t columns;
    int wide;                   // FP32
    int transposed;
    uint16_t* to;               // [rows, pitch], or transposed [columns, pitch]
    int64_t pitch;
    int tiles;                  // set by the launcher
};

struct FeedForwardPack {
    int count;
    PackMatrix matrices[5];
};

void plan_product(int64_t rows, int64_t columns, int64_t stages, FeedForwardProduct* a);
void plan_weights(FeedForwardWeights* a);
hipError_t launch_feed_forward_gate(const FeedForwardArgs& a, hipStream_t stream);
hipError_t launch_feed_forward_product(const FeedForwardProduct& a, hipStream_t stream);
hipError_t launch_feed_forward_grad(const FeedForwardArgs& a, hipStream_t stream);
hipError_t launch_feed_forward_weights(const FeedForwardWeights& a, hipStream_t stream);
hipError_t launch_feed_forward_join(const FeedForwardJoin& a, int outputs, hipStream_t stream);
hipError_t launch_feed_forward_pack(const FeedForwardPack& a, int type, hipStream_t stream);

// Rotary positions (lsso_rotary.hip).
struct RotaryTensor {
    const void* x;              // [batch, length, heads, features], unit feature stride
    void* y;                    // contiguous
    int64_t batch_stride;
    int64_t token_stride;
    int64_t head_stride;
    int heads;
};

struct RotaryArgs {
    RotaryTensor tensors[2];
    int count;
    int64_t batch;
    int64_t length;
    int features;
    int half;                   // pairs
    const double* frequencies;  // [half] radians a position
    float amplitude;
    float sign;                 // -1: turned back
    const void* positions;      // or nullptr: 0 .. length - 1
    int position_type;
    int64_t position_batch_stride;
    int64_t position_token_stride;
    int heads_each;             // heads of a workgroup, set by the launcher
};

hipError_t launch_rotary(const RotaryArgs& a, int dtype, int layout, hipStream_t stream);

// Group norm with an activation (lsso_group_norm.hip).
struct GroupNormArgs {
    const void* x;              // [samples, length, channels] contiguous
    int64_t samples;
    int64_t length;
    int channels;
    int groups;
    const void* weight;         // [channels] of parameter_type, or nullptr: ones
    const void* bias;           // [channels], or nullptr: zeros
    int parameter_type;
    float eps;
    int activation;             // 0, LSSO_HIP_SILU or LSSO_HIP_GELU
    const uint8_t* row_mask;    // [samples, length] or nullptr
    void* y;                    // contiguous
    float* statistics;          // [samples, groups, 2]: mean, 1 / sqrt(var + eps)
    const void* dy;             // of the backward, as what follows
    void* dx;                   // or nullptr
    void* grad_weight;          // [channels] of parameter_type, or nullptr
    void* grad_bias;
    float* partials;            // workspace
    float* sums;                // [samples, groups, 2]: mean of dn, mean of dn xhat
    int64_t splits;             // set by plan_group_norm: workgroups along the tokens of a sample
    int64_t split_rows;
    int team;                   // tokens are samples: lanes of a group, up to 64 or 256; 0: the kernels over splits
    int team_pieces;            // pieces of a lane
    int vector;                 // channels of a piece
    int64_t blocks;             // of the team kernel's grid
};

// Sets the plan; partial_bytes: of `partials`.
void plan_group_norm(GroupNormArgs* a, bool backward, size_t* partial_bytes);
hipError_t launch_group_norm(const GroupNormArgs& a, int dtype, hipStream_t stream);
hipError_t launch_group_norm_backward(const GroupNormArgs& a, int dtype, hipStream_t stream);

// Linear attention with a decay for each head (lsso_linear_attention.hip):
//   out_t = sum over s <= t of decay^(tokens from s to t) (a_t . b_s) c_s.
// A walk towards the front is the same with the last token's addresses and
// negative token strides.
struct WalkTensor {
    const void* data;
    int64_t batch;              // strides in elements
    int64_t token;
    int64_t head;
    int heads_per;              // heads of the walk that read one head of this tensor
};

struct WalkArgs {
    WalkTensor a;               // [batch, length, heads, features]
    WalkTensor b;
    WalkTensor c;               // [batch, length, heads, out_features]
    WalkTensor out;             // [batch, length, heads, out_features]; no data: the last state alone
    int wide_out;               // FP32, else of the inputs' type
    int64_t batch;
    int64_t length;
    int heads;
    int features;
    int out_features;
    const float* log_decay;     // [heads]
    const uint8_t* mask;        // or nullptr
    int64_t mask_batch;
    int64_t mask_token;
    float scale_within;         // of a_t . b_s
    float scale_across;         // of a_t . state
    float scale_update;         // of b_s (x) c_s
    int shift;                  // the first state counts from the first token, not from before it
    const float* first;         // [batch, heads, features, out_features] by these strides, or nullptr: zeros
    int64_t first_row;
    int64_t first_column;
    float* last;                // the state after the last token, contiguous, or nullptr
    float* updates;             // [batch, heads, pieces, features, out_features]: what each piece adds to the state
    int* counts;                // [batch, pieces] tokens that count
    float* states;              // [batch, heads, segments, features, out_features]: before each segment's first token
    int64_t states_row;         // their strides
    int64_t states_column;
    int reuse;                  // states are there already
    int64_t segment_chunks;     // set by plan_walk
    int64_t segments;
    int64_t piece_chunks;
    int64_t segment_pieces;     // of a segment, the last of them shorter
    int64_t pieces;             // of all segments but the last; 0 with one segment
};

constexpr int kWalkFeatures = 128;   // most features of a head
void plan_walk(WalkArgs* a);
hipError_t launch_walk(const WalkArgs& a, int dtype, hipStream_t stream);

// out[r, g, :] = sum over its `shared` heads of partial[r, g * shared + i, :].
struct HeadSumArgs {
    const float* partial;       // [rows, kv_heads * shared, features] contiguous
    void* out;                  // [rows, kv_heads, features] contiguous
    int64_t rows;
    int kv_heads;
    int shared;
    int features;
};
hipError_t launch_head_sum(const HeadSumArgs& a, int dtype, hipStream_t stream);

struct AttentionStepArgs {
    WalkTensor q;               // token strides unused
    WalkTensor k;
    WalkTensor v;
    void* y;                    // [batch, heads, value_features] contiguous
    int64_t batch;
    int heads;
    int features;
    int value_features;
    const float* log_decay;
    const uint8_t* mask;        // [batch] or nullptr
    float scale;
    float* state;               // [batch, heads, features, value_features], batch stride state_batch
    int64_t state_batch;
};
hipError_t launch_attention_step(const AttentionStepArgs& a, int dtype, hipStream_t stream);

// Sets the calling thread's error message (lsso_hip_last_error) and returns code.
int report(int code, const char* message) noexcept;
int report_hip(hipError_t error, const char* where) noexcept;

hipError_t launch_dropout(const DropoutArgs& a, int dtype, hipStream_t stream);
hipError_t launch_embedding(const EmbeddingArgs& a, int y_type, hipStream_t stream);
void plan_embedding_grad(EmbeddingArgs* a, size_t* bytes);
hipError_t launch_embedding_grad(const EmbeddingArgs& a, void* workspace, int grad_type, hipStream_t stream);

hipError_t launch_phase(const PhaseArgs& a, hipStream_t stream);
hipError_t launch_geometry(const GeometryArgs& a, int position_type, hipStream_t stream);
hipError_t launch_reduce(int rank, const ReduceArgs& a, int cpw, bool vec, hipStream_t stream);
// Heads per workgroup of the staged reduce for this geometry (items: samples x
// chunks) on a device of compute_units, or 0 where it does not apply (the
// one-wave-per-item reduce_kernel runs instead).
int64_t reduce_staged_group_heads(int64_t rank, int64_t heads, int64_t head_dim, int64_t column_groups,
                                  int64_t items, int64_t compute_units, bool vec);
hipError_t launch_solve(int rank, const SolveArgs& a, int64_t systems, hipStream_t stream);
hipError_t launch_apply(int rank, const ApplyArgs& a, int nfbw, bool vec, hipStream_t stream);
// Heads per workgroup of the staged apply for this geometry, or 0 where it
// does not apply.
int64_t apply_staged_group_heads(int64_t rank, int64_t heads, int64_t head_dim, int nfbw, bool vec);

// Projection launcher; k_steps = ceil(in_features / 16) rounded to a
// compiled tier.  Returns hipErrorInvalidValue for an unsupported tier.
// Shapes the fused apply + output projection handles: heads <= 8, head_dim a
// multiple of 16 up to 64, D = heads * head_dim <= 256, width <= 640.
bool mix_project_supported(int64_t rank, int64_t heads, int64_t head_dim, int64_t width);
int mix_project_tile_rows();
hipError_t launch_mix_project(int rank, const MixProjectArgs& a, int y_dtype, hipStream_t stream);

bool backward_supported(int64_t rank, int64_t head_dim);
// Record offsets (bf16 elements) of the token-map operands of one system;
// returns the per-system record size.
int64_t bwd_record_layout(int64_t rank, int64_t head_dim, int64_t* off_m, int64_t* off_e,
                          int64_t* off_g, int64_t* off_f, int* feature_k32);
hipError_t launch_bwd_solve(int rank, const BwdSolveArgs& a, int64_t systems, hipStream_t stream);
hipError_t launch_bwd_apply(int rank, const BwdApplyArgs& a, bool dk32, bool vec, hipStream_t stream);
// True when launch_bwd_apply runs the resident token map, which also writes
// column_part when it is set.
bool bwd_apply_resident(int rank, int64_t head_dim, bool vec);
hipError_t launch_column_sum(const float* partials, int64_t splits, int64_t cols, float* out,
                             hipStream_t stream);
// Two column sums over the same number of splits in one launch (partials2
// may be null when cols2 is 0).
hipError_t launch_column_sums(const float* partials, int64_t cols, float* out, const float* partials2,
                              int64_t cols2, float* out2, int64_t splits, hipStream_t stream);
hipError_t launch_param_reduce(const ParamReduceArgs& a, hipStream_t stream);

hipError_t launch_linear(const LinearArgs& a, int k_steps, int x_dtype, int y_dtype,
                         int grid_groups, hipStream_t stream);
// Heads per group of the fused projection + reduce for this geometry, or 0
// when the shape is outside the fused envelope.
int project_reduce_group_heads(int64_t rank, int64_t heads, int64_t head_dim,
                               int64_t in_features);
int project_reduce_tile_rows();
hipError_t launch_project_reduce(int rank, const ProjectReduceArgs& a, int x_dtype, int grid,
                                 hipStream_t stream);
// out[cols, rows] = in[rows, cols]^T of two FP32 matrices in one launch
// (either may be absent: rows 0).
hipError_t launch_transpose2(const float* in1, int64_t rows1, int64_t cols1, float* out1, const float* in2,
                             int64_t rows2, int64_t cols2, float* out2, hipStream_t stream);
hipError_t launch_grad_columns(const GradColumnsArgs& a, int g_dtype, bool vec, int64_t splits,
                               int64_t slabs, float* column_sums, hipStream_t stream);
void plan_weight_grad(int64_t rows, int64_t in_features, int64_t out_features, int64_t* splits,
                      int64_t* rows_per_split);
hipError_t launch_weight_grad(const WeightGradArgs& a, int g_dtype, int x_dtype, hipStream_t stream);
int linear_tile_rows(int k_steps);
int linear_columns_per_group(int k_steps);
int linear_k_tier(int64_t in_features);

}  // namespace lsso_hip
