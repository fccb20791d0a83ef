// staleynet_cuda.hpp — C++ host mirror of the reference's `staleynet-cuda` GEMM
// API, built on the C ABI in include/staleynet_gemm.h.
//
// Names, argument meaning and failure behaviour follow the Rust originals:
//   Storage, BatchStrides, MatmulSpec + builders   crates/staleynet-cuda/src/ops/matmul.rs:14-142
//   WriteMode                                      crates/staleynet-cuda/src/ops/mod.rs:251-269
//   MatmulKernel + tolerance                       crates/staleynet-cuda/src/device.rs:38-67
//   Gpu (new, bind, synchronize, zeros, upload,
//        download, copy_from_host, fill_zero)      crates/staleynet-cuda/src/device.rs:129-208
//   Gpu::matmul                                    crates/staleynet-cuda/src/ops/matmul.rs:144-171
//   Gpu::add_row_bias, Gpu::accumulate_column_sums crates/staleynet-cuda/src/ops/elementwise.rs:30-58
//   Gpu::matmul_bias (matmul + add_row_bias fused; no reference counterpart: the two calls of
//                     Linear::forward, crates/staleynet-model/src/layers/linear.rs:46-47)
//   Gpu::matmul_column_sums (matmul + accumulate_column_sums of the right operand fused; no
//                     reference counterpart: the two calls of Linear::backward,
//                     crates/staleynet-model/src/layers/linear.rs:54-59)
//   Shape, Tensor                                  crates/staleynet-cuda/src/device.rs:210-275
//   TokenBuffer, Gpu::upload_tokens                crates/staleynet-cuda/src/device.rs:35-36, :194-197
//   Gpu::causal_softmax, Gpu::softmax_backward     crates/staleynet-cuda/src/ops/attention.rs:54-92
//   HeadLayout, Gpu::split_heads / merge_heads     crates/staleynet-cuda/src/kernels/attention.rs:19-75,
//                                                  crates/staleynet-cuda/src/ops/attention.rs:10-52
//   CrossEntropyHead, Gpu::cross_entropy           crates/staleynet-cuda/src/ops/loss.rs:14-71
//   Gpu::causal_attention (scores, causal_softmax and mix in one launch; no reference counterpart:
//                     the three calls of crates/staleynet-model/src/layers/attention.rs:206-213)
//   Gpu::causal_attention_score_grad (the dP product and softmax_backward in one launch; no
//                     reference counterpart: crates/staleynet-model/src/layers/attention.rs:238-248)
//   Gpu::causal_attention_with_stats, Gpu::causal_attention_backward (the forward keeping per-query
//                     statistics instead of the probabilities, and the backward that recomputes
//                     them; no reference counterpart: layers/attention.rs:206-213 and :238-260)
//   ByteBuffer, Fp4Matrix, Fp4Cache, Gpu::quantize_fp4 / dequantize_fp4 / matmul_fp4 /
//   fp4_cache_append / fp4_cache_read / fp4_attention (4-bit weights and cache, staleynet_fp4.h; no
//                     reference counterpart)
//   Fp8Matrix, Gpu::quantize_fp8 / dequantize_fp8 / matmul_fp8 (8-bit operands, staleynet_fp8.h), Gpu::rms_norm /
//   rms_norm_fp8 / rms_norm_backward (staleynet_norm.h), Gpu::token_logprobs / token_logprobs_backward
//                     (staleynet_logprobs.h; no reference counterpart)
// The reference panics on undersized operands; here that is a thrown
// staleynet_cuda::Panic carrying the same message. Driver errors (the
// reference's Err(DriverError)) are thrown as staleynet_cuda::GpuError.
// `new` is a C++ keyword, so constructors named `new` in Rust are `new_`.
#pragma once

#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "staleynet_fp4.h"
#include "staleynet_fp8.h"
#include "staleynet_gemm.h"
#include "staleynet_logprobs.h"
#include "staleynet_norm.h"

namespace staleynet_cuda {

// An `assert!` of the reference, reported instead of aborting.
struct Panic : std::logic_error {
    int status;
    Panic(int code, const char* message) : std::logic_error(message), status(code) {}
};

// A runtime failure (`Err(DriverError)` in the reference).
struct GpuError : std::runtime_error {
    int status;
    explicit GpuError(int code) : std::runtime_error(sn_status_string(code)), status(code) {}
};

inline void check(int status) {
    if (status == SN_OK) return;
    if (status > 0 || status == SN_ERR_NO_DEVICE) throw GpuError(status);
    throw Panic(status, sn_status_string(status));
}

enum class Storage { RowMajor, Transposed };
enum class WriteMode { Overwrite, Accumulate };

// The reference's kernel choice. Naive and Tiled map to the reference-order
// kernel, Blocked to the fp32 matrix-core kernel (the default), TensorCore
// to the bf16-input matrix-core kernel that takes TF32's role on MI355X.
enum class MatmulKernel { Naive, Tiled, Blocked, TensorCore };

inline uint32_t abi_kernel(MatmulKernel kernel) {
    switch (kernel) {
        case MatmulKernel::Naive:
        case MatmulKernel::Tiled:
            return SN_KERNEL_SIMPLE;
        case MatmulKernel::Blocked:
            return SN_KERNEL_MFMA_F32;
        case MatmulKernel::TensorCore:
            return SN_KERNEL_MFMA_BF16;
    }
    return SN_KERNEL_MFMA_F32;
}

// `MatmulKernel::tolerance`: the largest relative error the kernel's arithmetic allows.
inline float tolerance(MatmulKernel kernel) { return sn_kernel_tolerance(abi_kernel(kernel)); }

inline const char* name(MatmulKernel kernel) {
    switch (kernel) {
        case MatmulKernel::Naive:
            return "Naive";
        case MatmulKernel::Tiled:
            return "Tiled";
        case MatmulKernel::Blocked:
            return "Blocked";
        case MatmulKernel::TensorCore:
            return "TensorCore";
    }
    return "?";
}

struct BatchStrides {
    size_t count;
    size_t left;
    size_t right;
    size_t output;
    static constexpr BatchStrides single() { return BatchStrides{1, 0, 0, 0}; }
};

struct MatmulSpec {
    size_t rows = 0;
    size_t cols = 0;
    size_t inner = 0;
    Storage left = Storage::RowMajor;
    Storage right = Storage::RowMajor;
    BatchStrides batch = BatchStrides::single();
    float scale = 1.0f;
    WriteMode write = WriteMode::Overwrite;
    // Extensions (no reference counterpart; zero keeps the reference's behaviour).
    uint32_t mask = SN_MASK_NONE;
    size_t query_offset = 0;

    static MatmulSpec new_(size_t rows, size_t cols, size_t inner) {
        MatmulSpec spec;
        spec.rows = rows;
        spec.cols = cols;
        spec.inner = inner;
        return spec;
    }
    MatmulSpec left_transposed() const { MatmulSpec s = *this; s.left = Storage::Transposed; return s; }
    MatmulSpec right_transposed() const { MatmulSpec s = *this; s.right = Storage::Transposed; return s; }
    MatmulSpec accumulate() const { MatmulSpec s = *this; s.write = WriteMode::Accumulate; return s; }
    MatmulSpec scaled(float factor) const { MatmulSpec s = *this; s.scale = factor; return s; }
    MatmulSpec batched(BatchStrides strides) const { MatmulSpec s = *this; s.batch = strides; return s; }
    MatmulSpec causal_output(size_t offset) const {
        MatmulSpec s = *this;
        s.mask = SN_MASK_CAUSAL_OUTPUT;
        s.query_offset = offset;
        return s;
    }
    MatmulSpec causal_left(size_t offset) const {
        MatmulSpec s = *this;
        s.mask = SN_MASK_CAUSAL_LEFT;
        s.query_offset = offset;
        return s;
    }

    // Elements an operand of `per_matrix` elements must hold (ops/matmul.rs:139-141).
    size_t required_len(size_t stride, size_t per_matrix) const { return (batch.count - 1) * stride + per_matrix; }

    sn_matmul_spec to_ffi() const {
        sn_matmul_spec c = sn_matmul_spec_new(rows, cols, inner);
        c.left_storage = left == Storage::Transposed ? SN_TRANSPOSED : SN_ROW_MAJOR;
        c.right_storage = right == Storage::Transposed ? SN_TRANSPOSED : SN_ROW_MAJOR;
        c.batch_count = batch.count;
        c.batch_left = batch.left;
        c.batch_right = batch.right;
        c.batch_output = batch.output;
        c.scale = scale;
        c.write = write == WriteMode::Accumulate ? SN_ACCUMULATE : SN_OVERWRITE;
        c.mask = mask;
        c.query_offset = query_offset;
        return c;
    }
};

struct Shape {
    size_t rows;
    size_t cols;
    static constexpr Shape new_(size_t rows, size_t cols) { return Shape{rows, cols}; }
    static constexpr Shape vector(size_t cols) { return Shape{1, cols}; }
    constexpr size_t len() const { return rows * cols; }
    constexpr bool is_empty() const { return len() == 0; }
};

// A row-major f32 matrix in device memory; owns its buffer (move-only).
class Tensor {
   public:
    Tensor() = default;
    Tensor(sn_context* context, float* buffer, Shape shape) : context_(context), buffer_(buffer), shape_(shape) {}
    Tensor(const Tensor&) = delete;
    Tensor& operator=(const Tensor&) = delete;
    Tensor(Tensor&& other) noexcept { *this = std::move(other); }
    Tensor& operator=(Tensor&& other) noexcept {
        if (this != &other) {
            release();
            context_ = std::exchange(other.context_, nullptr);
            buffer_ = std::exchange(other.buffer_, nullptr);
            shape_ = other.shape_;
        }
        return *this;
    }
    ~Tensor() { release(); }

    Shape shape() const { return shape_; }
    size_t len() const { return shape_.len(); }
    bool is_empty() const { return shape_.is_empty(); }
    const float* data() const { return buffer_; }
    float* data() { return buffer_; }

   private:
    void release() {
        if (buffer_ != nullptr) sn_free(context_, buffer_);
        buffer_ = nullptr;
    }
    sn_context* context_ = nullptr;
    float* buffer_ = nullptr;
    Shape shape_{0, 0};
};

// Token ids (u32) in device memory; owns its buffer (move-only).
class TokenBuffer {
   public:
    TokenBuffer() = default;
    TokenBuffer(sn_context* context, uint32_t* buffer, size_t count) : context_(context), buffer_(buffer), count_(count) {}
    TokenBuffer(const TokenBuffer&) = delete;
    TokenBuffer& operator=(const TokenBuffer&) = delete;
    TokenBuffer(TokenBuffer&& other) noexcept { *this = std::move(other); }
    TokenBuffer& operator=(TokenBuffer&& other) noexcept {
        if (this != &other) {
            release();
            context_ = std::exchange(other.context_, nullptr);
            buffer_ = std::exchange(other.buffer_, nullptr);
            count_ = std::exchange(other.count_, 0);
        }
        return *this;
    }
    ~TokenBuffer() { release(); }

    size_t len() const { return count_; }
    const uint32_t* data() const { return buffer_; }
    uint32_t* data() { return buffer_; }

   private:
    void release() {
        if (buffer_ != nullptr) sn_free_tokens(context_, buffer_);
        buffer_ = nullptr;
    }
    sn_context* context_ = nullptr;
    uint32_t* buffer_ = nullptr;
    size_t count_ = 0;
};

// Bytes in device memory: the codes or the scales of 4-bit or 8-bit blocks; owns its buffer (move-only).
class ByteBuffer {
   public:
    ByteBuffer() = default;
    ByteBuffer(sn_context* context, uint8_t* buffer, size_t count) : context_(context), buffer_(buffer), count_(count) {}
    ByteBuffer(const ByteBuffer&) = delete;
    ByteBuffer& operator=(const ByteBuffer&) = delete;
    ByteBuffer(ByteBuffer&& other) noexcept { *this = std::move(other); }
    ByteBuffer& operator=(ByteBuffer&& other) noexcept {
        if (this != &other) {
            release();
            context_ = std::exchange(other.context_, nullptr);
            buffer_ = std::exchange(other.buffer_, nullptr);
            count_ = std::exchange(other.count_, 0);
        }
        return *this;
    }
    ~ByteBuffer() { release(); }

    size_t len() const { return count_; }
    const uint8_t* data() const { return buffer_; }
    uint8_t* data() { return buffer_; }

   private:
    void release() {
        if (buffer_ != nullptr) sn_free_bytes(context_, buffer_);
        buffer_ = nullptr;
    }
    sn_context* context_ = nullptr;
    uint8_t* buffer_ = nullptr;
    size_t count_ = 0;
};

// A product's right operand [inner, cols] in 4 bits (staleynet_fp4.h).
struct Fp4Matrix {
    size_t cols = 0, inner = 0;
    ByteBuffer codes, scales;
};

// An operand of a product in 8 bits: `rows` rows of `inner` values (staleynet_fp8.h).
struct Fp8Matrix {
    size_t rows = 0, inner = 0;
    ByteBuffer codes, scales;
};

// A key/value cache [batch][kv_heads][capacity][head_dim] in 4 bits (staleynet_fp4.h).
struct Fp4Cache {
    sn_fp4_cache_shape shape{};
    ByteBuffer k_codes, k_scales, v_codes, v_scales;
};

// Where a group of attention heads sits in the packed activations and in the
// head-major tensor (HeadLayout, kernels/attention.rs:19-75).
struct HeadLayout {
    size_t batch, time, heads, head_dim, width, column_offset, time_capacity, time_offset;

    static HeadLayout dense(size_t batch, size_t time, size_t heads, size_t head_dim, size_t width,
                            size_t column_offset) {
        return HeadLayout{batch, time, heads, head_dim, width, column_offset, time, 0};
    }
    HeadLayout in_cache(size_t capacity, size_t offset) const {
        HeadLayout l = *this;
        l.time_capacity = capacity;
        l.time_offset = offset;
        return l;
    }
    size_t element_count() const { return batch * heads * time * head_dim; }
    sn_head_layout to_ffi() const {
        return sn_head_layout{batch, time, heads, head_dim, width, column_offset, time_capacity, time_offset};
    }
};

// Which columns of a logits row and which target of a target row one
// classifier owns (CrossEntropyHead, ops/loss.rs:14-30).
struct CrossEntropyHead {
    size_t column_offset, classes, target_stride, target_offset;
    float grad_scale;
};

// One device, one stream, and the kernel choice (device.rs:129-155).
class Gpu {
   public:
    // Public like the reference's field (device.rs:144); read on every matmul.
    MatmulKernel matmul_kernel = MatmulKernel::Blocked;

    static Gpu new_(int ordinal) {
        sn_context* context = nullptr;
        check(sn_context_create(ordinal, &context));
        return Gpu(context);
    }
    Gpu(Gpu&& other) noexcept : matmul_kernel(other.matmul_kernel), context_(std::exchange(other.context_, nullptr)) {}
    Gpu(const Gpu&) = delete;
    Gpu& operator=(const Gpu&) = delete;
    ~Gpu() {
        if (context_ != nullptr) sn_context_destroy(context_);
    }

    void bind_to_current_thread() const { check(sn_context_bind(context_)); }
    void synchronize() const { check(sn_synchronize(context_)); }

    Tensor zeros(Shape shape) const {
        float* buffer = nullptr;
        check(sn_alloc_zeroed(context_, shape.len(), &buffer));
        return Tensor(context_, buffer, shape);
    }

    Tensor upload(Shape shape, const std::vector<float>& values) const {
        if (values.size() != shape.len()) throw Panic(SN_ERR_UNSUPPORTED, "upload: value count does not match the shape");
        float* buffer = nullptr;
        check(sn_upload(context_, values.data(), values.size(), &buffer));
        return Tensor(context_, buffer, shape);
    }

    std::vector<float> download(const Tensor& tensor) const {
        std::vector<float> host(tensor.len());
        check(sn_download(context_, tensor.data(), host.size(), host.data()));
        return host;
    }

    void copy_from_host(Tensor& tensor, const std::vector<float>& values) const {
        if (values.size() != tensor.len()) throw Panic(SN_ERR_UNSUPPORTED, "copy_from_host: length mismatch");
        check(sn_copy_from_host(context_, tensor.data(), values.data(), values.size()));
    }

    void fill_zero(Tensor& tensor) const { check(sn_fill_zero(context_, tensor.data(), tensor.len())); }

    // `Gpu::matmul`: enqueue output = scale·op(left)·op(right) (+ output).
    void matmul(const MatmulSpec& spec, const Tensor& left, const Tensor& right, Tensor& output) const {
        check(sn_context_set_kernel(context_, abi_kernel(matmul_kernel)));
        const sn_matmul_spec c = spec.to_ffi();
        check(sn_matmul(context_, &c, left.data(), left.len(), right.data(), right.len(), output.data(),
                        output.len()));
    }

    // `Gpu::add_row_bias`: output[r, c] += bias[c].
    void add_row_bias(Tensor& output, const Tensor& bias) const {
        const int rc = sn_add_row_bias(context_, output.data(), output.shape().rows, output.shape().cols, bias.data(),
                                       bias.len());
        if (rc == SN_ERR_LENGTH_MISMATCH) throw Panic(rc, "add_row_bias: bias length must equal output columns");
        check(rc);
    }

    // `Gpu::accumulate_column_sums`: sums += the column sums of input.
    void accumulate_column_sums(const Tensor& input, Tensor& sums) const {
        const int rc = sn_accumulate_column_sums(context_, input.data(), input.shape().rows, input.shape().cols,
                                                 sums.data(), sums.len());
        if (rc == SN_ERR_LENGTH_MISMATCH)
            throw Panic(rc, "accumulate_column_sums: sums length must equal input columns");
        check(rc);
    }

    // `matmul` then `add_row_bias` on its output, in one pass (sn_matmul_bias).
    void matmul_bias(const MatmulSpec& spec, const Tensor& left, const Tensor& right, const Tensor& bias,
                     Tensor& output) const {
        check(sn_context_set_kernel(context_, abi_kernel(matmul_kernel)));
        const sn_matmul_spec c = spec.to_ffi();
        check(sn_matmul_bias(context_, &c, left.data(), left.len(), right.data(), right.len(), bias.data(),
                             bias.len(), output.data(), output.len()));
    }

    // `matmul` then `accumulate_column_sums(right, sums)`, in one call (sn_matmul_column_sums; the
    // right operand row-major, the spec unbatched).
    void matmul_column_sums(const MatmulSpec& spec, const Tensor& left, const Tensor& right, Tensor& output,
                            Tensor& sums) const {
        check(sn_context_set_kernel(context_, abi_kernel(matmul_kernel)));
        const sn_matmul_spec c = spec.to_ffi();
        check(sn_matmul_column_sums(context_, &c, left.data(), left.len(), right.data(), right.len(), output.data(),
                                    output.len(), sums.data(), sums.len()));
    }

    TokenBuffer upload_tokens(const std::vector<uint32_t>& tokens) const {
        uint32_t* buffer = nullptr;
        check(sn_upload_tokens(context_, tokens.data(), tokens.size(), &buffer));
        return TokenBuffer(context_, buffer, tokens.size());
    }

    std::vector<uint32_t> download_tokens(const TokenBuffer& tokens) const {
        std::vector<uint32_t> host(tokens.len());
        check(sn_download_tokens(context_, tokens.data(), host.size(), host.data()));
        return host;
    }

    // `Gpu::causal_softmax`: in place on [matrices · queries, keys] scores.
    void causal_softmax(Tensor& scores, size_t queries, float scale, size_t query_offset) const {
        const int rc = sn_causal_softmax(context_, scores.data(), scores.shape().rows, scores.shape().cols, queries,
                                         scale, query_offset);
        if (rc == SN_ERR_SHAPE) throw Panic(rc, "causal_softmax: rows must be a multiple of queries");
        check(rc);
    }

    // `Gpu::softmax_backward`: grad <- p * (grad - sum(grad * p)) per row.
    void softmax_backward(const Tensor& probabilities, Tensor& grad) const {
        const int rc = sn_softmax_backward(context_, probabilities.data(), probabilities.shape().rows,
                                           probabilities.shape().cols, grad.data(), grad.shape().rows,
                                           grad.shape().cols);
        if (rc == SN_ERR_SHAPE) throw Panic(rc, "softmax_backward: shape mismatch");
        check(rc);
    }

    // `Gpu::split_heads`: packed columns -> head-major tensor.
    void split_heads(const Tensor& packed, Tensor& head_major, const HeadLayout& layout) const {
        check_layout(layout, packed, head_major);
        const sn_head_layout l = layout.to_ffi();
        check(sn_split_heads(context_, packed.data(), packed.len(), head_major.data(), head_major.len(), &l));
    }

    // `Gpu::merge_heads`: head-major tensor -> packed columns (the others left alone).
    void merge_heads(const Tensor& head_major, Tensor& packed, const HeadLayout& layout) const {
        check_layout(layout, packed, head_major);
        const sn_head_layout l = layout.to_ffi();
        check(sn_merge_heads(context_, head_major.data(), head_major.len(), packed.data(), packed.len(), &l));
    }

    // `Gpu::cross_entropy`: one codebook's losses and its columns of the gradient.
    void cross_entropy(const Tensor& logits, const TokenBuffer& targets, const CrossEntropyHead& head, Tensor& losses,
                       Tensor& logits_grad) const {
        const Shape shape = logits.shape();
        if (logits_grad.shape().rows != shape.rows || logits_grad.shape().cols != shape.cols)
            throw Panic(SN_ERR_SHAPE, "cross_entropy: gradient shape");
        if (head.column_offset + head.classes > shape.cols) throw Panic(SN_ERR_SHAPE, "cross_entropy: head exceeds logits");
        if (losses.len() < shape.rows) throw Panic(SN_ERR_LENGTH_MISMATCH, "cross_entropy: losses too small");
        if (targets.len() < shape.rows * head.target_stride)
            throw Panic(SN_ERR_LENGTH_MISMATCH, "cross_entropy: too few targets");
        const sn_cross_entropy_head h{head.column_offset, head.classes, head.target_stride, head.target_offset,
                                      head.grad_scale};
        check(sn_cross_entropy(context_, logits.data(), shape.rows, shape.cols, targets.data(), targets.len(), &h,
                               losses.data(), losses.len(), logits_grad.data(), logits_grad.shape().rows,
                               logits_grad.shape().cols));
    }

    // The scores product, causal_softmax and the mix product in one launch
    // (sn_causal_attention); `probabilities` may be null.
    void causal_attention(const Tensor& q, const Tensor& k, const Tensor& v, Tensor& out, const sn_attention_shape& shape,
                          Tensor* probabilities = nullptr) const {
        check(sn_causal_attention(context_, &shape, q.data(), q.len(), k.data(), k.len(), v.data(), v.len(),
                                  out.data(), out.len(), probabilities ? probabilities->data() : nullptr,
                                  probabilities ? probabilities->len() : 0));
    }

    // The dP product and softmax_backward of the attention backward in one launch
    // (sn_causal_attention_score_grad): grad = P * (dO V^T - rowsum(dO * O)).
    // With k and q_grad, also the query gradient q_grad = shape.scale * grad K.
    void causal_attention_score_grad(const Tensor& d_out, const Tensor& v, const Tensor& out, const Tensor& probabilities,
                                     Tensor& grad, const sn_attention_shape& shape, const Tensor* k = nullptr,
                                     Tensor* q_grad = nullptr) const {
        check(sn_causal_attention_score_grad(context_, &shape, d_out.data(), d_out.len(), v.data(), v.len(),
                                             out.data(), out.len(), probabilities.data(), probabilities.len(),
                                             grad.data(), grad.len(), k ? k->data() : nullptr, k ? k->len() : 0,
                                             q_grad ? q_grad->data() : nullptr, q_grad ? q_grad->len() : 0));
    }

    // The fused forward keeping, per query, the maximum m of its scaled visible scores and the sum
    // l of e^(x - m) (2 floats, in `stats`) instead of the probabilities
    // (sn_causal_attention_with_stats); `out` is causal_attention's O.
    void causal_attention_with_stats(const Tensor& q, const Tensor& k, const Tensor& v, Tensor& out, Tensor& stats,
                                     const sn_attention_shape& shape) const {
        check(sn_causal_attention_with_stats(context_, &shape, q.data(), q.len(), k.data(), k.len(), v.data(), v.len(),
                                             out.data(), out.len(), stats.data(), stats.len()));
    }

    // The attention backward from O, dO and those statistics (sn_causal_attention_backward): the
    // query, key and value gradients CausalSelfAttention::backward leaves, with no P or dS in memory.
    void causal_attention_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                                   const Tensor& d_out, const Tensor& stats, Tensor& q_grad, Tensor& k_grad,
                                   Tensor& v_grad, const sn_attention_shape& shape) const {
        check(sn_causal_attention_backward(context_, &shape, q.data(), q.len(), k.data(), k.len(), v.data(), v.len(),
                                           out.data(), out.len(), d_out.data(), d_out.len(), stats.data(), stats.len(),
                                           q_grad.data(), q_grad.len(), k_grad.data(), k_grad.len(), v_grad.data(),
                                           v_grad.len()));
    }

    // Zeroed bytes (sn_alloc_bytes), and the 4-bit operands made of them.
    ByteBuffer zeros_bytes(size_t count) const {
        uint8_t* buffer = nullptr;
        check(sn_alloc_bytes(context_, count, &buffer));
        return ByteBuffer(context_, buffer, count);
    }
    Fp4Matrix fp4_matrix(size_t cols, size_t inner) const {
        size_t codes = 0, scales = 0;
        check(sn_fp4_sizes(cols, inner, &codes, &scales));
        return Fp4Matrix{cols, inner, zeros_bytes(codes), zeros_bytes(scales)};
    }
    Fp4Cache fp4_cache(const sn_fp4_cache_shape& shape) const {
        size_t rows = 0, codes = 0, scales = 0;
        if (__builtin_mul_overflow(shape.batch, shape.kv_heads, &rows) ||
            __builtin_mul_overflow(rows, shape.capacity, &rows))
            check(SN_ERR_OVERFLOW);
        check(sn_fp4_sizes(rows, shape.head_dim, &codes, &scales));
        return Fp4Cache{shape, zeros_bytes(codes), zeros_bytes(scales), zeros_bytes(codes), zeros_bytes(scales)};
    }

    // A right operand [inner, cols], stored as `storage` says, to 4 bits and back (sn_quantize_fp4,
    // sn_dequantize_fp4).
    void quantize_fp4(const Tensor& source, Fp4Matrix& matrix, Storage storage = Storage::RowMajor) const {
        check(sn_quantize_fp4(context_, matrix.cols, matrix.inner, abi_storage(storage), source.data(), source.len(),
                              matrix.codes.data(), matrix.codes.len(), matrix.scales.data(), matrix.scales.len()));
    }
    void dequantize_fp4(const Fp4Matrix& matrix, Tensor& output, Storage storage = Storage::RowMajor) const {
        check(sn_dequantize_fp4(context_, matrix.cols, matrix.inner, abi_storage(storage), matrix.codes.data(),
                                matrix.codes.len(), matrix.scales.data(), matrix.scales.len(), output.data(),
                                output.len()));
    }

    // `Gpu::matmul`, or with a bias matmul_bias, against a 4-bit right operand (sn_matmul_fp4); the spec
    // is right_transposed.
    void matmul_fp4(const MatmulSpec& spec, const Tensor& left, const Fp4Matrix& right, Tensor& output,
                    const Tensor* bias = nullptr) const {
        if (right.cols != spec.cols || right.inner != spec.inner)
            throw Panic(SN_ERR_RIGHT_TOO_SMALL, "matmul_fp4: the operand's columns and inner length are not the spec's");
        const sn_matmul_spec c = spec.to_ffi();
        check(sn_matmul_fp4(context_, &c, left.data(), left.len(), right.codes.data(), right.codes.len(),
                            right.scales.data(), right.scales.len(), bias ? bias->data() : nullptr,
                            bias ? bias->len() : 0, output.data(), output.len()));
    }

    // split_heads of the keys and values of packed rows into a 4-bit cache, at each sequence's own
    // position where `positions` is given (sn_fp4_cache_append), and their values (sn_fp4_cache_read).
    void fp4_cache_append(Fp4Cache& cache, const sn_fp4_cache_rows& rows, const Tensor& packed,
                          const TokenBuffer* positions = nullptr) const {
        check(sn_fp4_cache_append(context_, &cache.shape, &rows, packed.data(), packed.len(),
                                  positions ? positions->data() : nullptr, positions ? positions->len() : 0,
                                  cache.k_codes.data(), cache.k_codes.len(), cache.k_scales.data(),
                                  cache.k_scales.len(), cache.v_codes.data(), cache.v_codes.len(),
                                  cache.v_scales.data(), cache.v_scales.len()));
    }
    void fp4_cache_read(const Fp4Cache& cache, const sn_fp4_cache_rows& rows, Tensor& keys, Tensor& values,
                        const TokenBuffer* positions = nullptr) const {
        check(sn_fp4_cache_read(context_, &cache.shape, &rows, cache.k_codes.data(), cache.k_codes.len(),
                                cache.k_scales.data(), cache.k_scales.len(), cache.v_codes.data(),
                                cache.v_codes.len(), cache.v_scales.data(), cache.v_scales.len(),
                                positions ? positions->data() : nullptr, positions ? positions->len() : 0,
                                keys.data(), keys.len(), values.data(), values.len()));
    }

    // Causal attention over a 4-bit cache (sn_fp4_attention); `lengths` null: shape.keys for every sequence.
    void fp4_attention(const Fp4Cache& cache, const sn_fp4_attention_shape& shape, const Tensor& q, Tensor& out,
                       const TokenBuffer* lengths = nullptr) const {
        check(sn_fp4_attention(context_, &cache.shape, &shape, q.data(), q.len(), cache.k_codes.data(),
                               cache.k_codes.len(), cache.k_scales.data(), cache.k_scales.len(),
                               cache.v_codes.data(), cache.v_codes.len(), cache.v_scales.data(),
                               cache.v_scales.len(), lengths ? lengths->data() : nullptr,
                               lengths ? lengths->len() : 0, out.data(), out.len()));
    }

    Fp8Matrix fp8_matrix(size_t rows, size_t inner) const {
        size_t codes = 0, scales = 0;
        check(sn_fp8_sizes(rows, inner, &codes, &scales));
        return Fp8Matrix{rows, inner, zeros_bytes(codes), zeros_bytes(scales)};
    }

    // An operand to 8 bits and back, stored as `storage` says: [rows, inner], or a weight's [inner, rows]
    // (sn_quantize_fp8, sn_dequantize_fp8).
    void quantize_fp8(const Tensor& source, Fp8Matrix& matrix, Storage storage = Storage::RowMajor) const {
        check(sn_quantize_fp8(context_, matrix.rows, matrix.inner, abi_storage(storage), source.data(), source.len(),
                              matrix.codes.data(), matrix.codes.len(), matrix.scales.data(), matrix.scales.len()));
    }
    void dequantize_fp8(const Fp8Matrix& matrix, Tensor& output, Storage storage = Storage::RowMajor) const {
        check(sn_dequantize_fp8(context_, matrix.rows, matrix.inner, abi_storage(storage), matrix.codes.data(),
                                matrix.codes.len(), matrix.scales.data(), matrix.scales.len(), output.data(),
                                output.len()));
    }

    // `Gpu::matmul`, or with a bias matmul_bias, of two 8-bit operands (sn_matmul_fp8); the spec is right_transposed.
    void matmul_fp8(const MatmulSpec& spec, const Fp8Matrix& left, const Fp8Matrix& right, Tensor& output,
                    const Tensor* bias = nullptr) const {
        if (left.rows != spec.rows || left.inner != spec.inner)
            throw Panic(SN_ERR_LEFT_TOO_SMALL, "matmul_fp8: the left operand's rows and inner length are not the spec's");
        if (right.rows != spec.cols || right.inner != spec.inner)
            throw Panic(SN_ERR_RIGHT_TOO_SMALL, "matmul_fp8: the right operand's columns and inner length are not the spec's");
        const sn_matmul_spec c = spec.to_ffi();
        check(sn_matmul_fp8(context_, &c, left.codes.data(), left.codes.len(), left.scales.data(), left.scales.len(),
                            right.codes.data(), right.codes.len(), right.scales.data(), right.scales.len(),
                            bias ? bias->data() : nullptr, bias ? bias->len() : 0, output.data(), output.len()));
    }

    // sum = x + residual and out = its root-mean-square norm (sn_rms_norm); residual, sum and inverse may be null, and
    // sum may be x or residual.
    void rms_norm(const sn_rms_norm_shape& shape, const Tensor& x, const Tensor* residual, const Tensor& weight,
                  Tensor* sum, Tensor& out, Tensor* inverse = nullptr) const {
        check(sn_rms_norm(context_, &shape, x.data(), x.len(), data_of(residual), len_of(residual), weight.data(),
                          weight.len(), data_of(sum), len_of(sum), out.data(), out.len(), data_of(inverse),
                          len_of(inverse)));
    }
    // The same rounded to 8-bit rows (sn_rms_norm_fp8).
    void rms_norm_fp8(const sn_rms_norm_shape& shape, const Tensor& x, const Tensor* residual, const Tensor& weight,
                      Tensor* sum, Fp8Matrix& out) const {
        if (out.rows != shape.rows || out.inner != shape.width)
            throw Panic(SN_ERR_LENGTH_MISMATCH, "rms_norm_fp8: the 8-bit rows are not the shape's");
        check(sn_rms_norm_fp8(context_, &shape, x.data(), x.len(), data_of(residual), len_of(residual), weight.data(),
                              weight.len(), data_of(sum), len_of(sum), out.codes.data(), out.codes.len(),
                              out.scales.data(), out.scales.len()));
    }
    // The norm's gradients (sn_rms_norm_backward); d_sum and d_weight may be null, and d_x may be d_sum.
    void rms_norm_backward(const sn_rms_norm_shape& shape, const Tensor& sum, const Tensor& inverse,
                           const Tensor& weight, const Tensor& d_out, const Tensor* d_sum, Tensor& d_x,
                           Tensor* d_weight) const {
        check(sn_rms_norm_backward(context_, &shape, sum.data(), sum.len(), inverse.data(), inverse.len(),
                                   weight.data(), weight.len(), d_out.data(), d_out.len(), data_of(d_sum),
                                   len_of(d_sum), d_x.data(), d_x.len(), data_of(d_weight), len_of(d_weight)));
    }

    // Log probabilities of tokens, entropies, the backward's stats and the likeliest classes (sn_token_logprobs), each
    // where it is given.
    void token_logprobs(const sn_logprob_shape& shape, const Tensor& logits, const TokenBuffer* tokens,
                        Tensor* logprobs, Tensor* entropies, Tensor* stats, TokenBuffer* top_tokens = nullptr,
                        Tensor* top_logprobs = nullptr) const {
        check(sn_token_logprobs(context_, &shape, logits.data(), logits.len(), tokens ? tokens->data() : nullptr,
                                tokens ? tokens->len() : 0, data_of(logprobs), len_of(logprobs), data_of(entropies),
                                len_of(entropies), data_of(stats), len_of(stats),
                                top_tokens ? top_tokens->data() : nullptr, top_tokens ? top_tokens->len() : 0,
                                data_of(top_logprobs), len_of(top_logprobs)));
    }
    // The gradient of the logits (sn_token_logprobs_backward); it may be the logits themselves.
    void token_logprobs_backward(const sn_logprob_shape& shape, const Tensor& logits, const TokenBuffer* tokens,
                                 const Tensor& stats, const Tensor* entropies, const Tensor* d_logprobs,
                                 const Tensor* d_entropies, Tensor& grad) const {
        check(sn_token_logprobs_backward(context_, &shape, logits.data(), logits.len(),
                                         tokens ? tokens->data() : nullptr, tokens ? tokens->len() : 0, stats.data(),
                                         stats.len(), data_of(entropies), len_of(entropies), data_of(d_logprobs),
                                         len_of(d_logprobs), data_of(d_entropies), len_of(d_entropies), grad.data(),
                                         grad.len()));
    }

    sn_context* raw() const { return context_; }

   private:
    static const float* data_of(const Tensor* t) { return t ? t->data() : nullptr; }
    static float* data_of(Tensor* t) { return t ? t->data() : nullptr; }
    static size_t len_of(const Tensor* t) { return t ? t->len() : 0; }

    static uint32_t abi_storage(Storage storage) {
        return storage == Storage::Transposed ? SN_TRANSPOSED : SN_ROW_MAJOR;
    }

    // check_layout (ops/attention.rs:11-18).
    static void check_layout(const HeadLayout& layout, const Tensor& packed, const Tensor& head_major) {
        if (layout.time_offset + layout.time > layout.time_capacity)
            throw Panic(SN_ERR_SHAPE, "HeadLayout: time range exceeds capacity");
        if (packed.len() < layout.batch * layout.time * layout.width)
            throw Panic(SN_ERR_LENGTH_MISMATCH, "HeadLayout: packed tensor too small");
        if (head_major.len() < layout.batch * layout.heads * layout.time_capacity * layout.head_dim)
            throw Panic(SN_ERR_LENGTH_MISMATCH, "HeadLayout: head-major tensor too small");
    }

    explicit Gpu(sn_context* context) : context_(context) {}
    sn_context* context_ = nullptr;
};

}  // namespace staleynet_cuda
