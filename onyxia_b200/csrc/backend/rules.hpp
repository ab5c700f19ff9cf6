// The rules of a batch of requests on the logits of their next tokens, as tensors of the device, and what is wrong with them.
#pragma once
#include "runtime.hpp"

namespace oxrt {

// Row r of every tensor belongs to row r of the logits; null: no such rule.
struct Rules {
    const DTensor* history = nullptr;    // I32 [rows, width]: the tokens of the prompt, then those of the answer
    const DTensor* lengths = nullptr;    // I32 [rows, 2]: how many of them are the prompt's, how many there are
    const DTensor* penalties = nullptr;  // F32 [rows, 3]: repetition, frequency, presence
    const DTensor* bias_ids = nullptr;   // I32 [rows, n]; negative: none
    const DTensor* bias = nullptr;       // F32 [rows, n]
    const DTensor* masks = nullptr;      // U32 [n, ⌈vocab / 32⌉]: a set bit allows a token, the lowest bit of a word the first
    const DTensor* mask_of = nullptr;    // I32 [rows]: the row's mask; negative: none. Null: row r has mask r
};
constexpr int64_t kMaxBiases = 4096;

inline void check_rules(const DTensor& logits, const Rules& r) {
    using ox::ErrKind;
    using ox::fail;
    if ((logits.dtype != DType::F32 && logits.dtype != DType::F16) || logits.shape.empty() || logits.shape.back() == 0 || !logits.buf)
        fail(ErrKind::DType, "rules need an f32 or f16 tensor with a non-empty last axis");
    if (logits.cap != 0) fail(ErrKind::Shape, "rules: logits must be densely packed");
    const int64_t cols = logits.shape.back(), rows = logits.numel() / cols;
    if (cols > INT32_MAX || rows > 65535) fail(ErrKind::Shape, "rules: at most 65535 rows of 2^31 - 1 logits");
    auto is = [&](const DTensor* t, const char* name, DType dtype, int64_t dim0, int64_t dim1) {  // −1: any
        if (t->dtype != dtype) fail(ErrKind::DType, std::string("rules: ") + name + " must be " + dtype_name(dtype));
        const size_t rank = dim1 == 0 ? 1 : 2;
        if (!t->buf || t->cap != 0 || t->shape.size() != rank || (dim0 >= 0 && t->shape[0] != dim0) || (rank == 2 && dim1 > 0 && t->shape[1] != dim1))
            fail(ErrKind::Shape, std::string("rules: ") + name + " has the wrong shape");
    };
    if (!r.history != !r.lengths || !r.history != !r.penalties) fail(ErrKind::Shape, "rules: history, lengths and penalties come together");
    if (!r.bias_ids != !r.bias) fail(ErrKind::Shape, "rules: bias_ids and bias come together");
    if (r.mask_of && !r.masks) fail(ErrKind::Shape, "rules: mask_of without masks");
    if (r.history) {
        is(r.history, "history", DType::I32, rows, -1);
        is(r.lengths, "lengths", DType::I32, rows, 2);
        is(r.penalties, "penalties", DType::F32, rows, 3);
        if (r.history->shape[1] > INT32_MAX) fail(ErrKind::Shape, "rules: history has the wrong shape");
    }
    if (r.bias_ids) {
        is(r.bias_ids, "bias_ids", DType::I32, rows, -1);
        is(r.bias, "bias", DType::F32, rows, r.bias_ids->shape[1] ? r.bias_ids->shape[1] : -1);
        if (r.bias->shape != r.bias_ids->shape) fail(ErrKind::Shape, "rules: bias has the wrong shape");
        if (r.bias_ids->shape[1] > kMaxBiases) fail(ErrKind::Shape, "rules: at most " + std::to_string(kMaxBiases) + " biases of a row");
    }
    if (r.masks) {
        is(r.masks, "masks", DType::U32, r.mask_of ? -1 : rows, (cols + 31) / 32);
        if (r.masks->shape[0] > INT32_MAX) fail(ErrKind::Shape, "rules: masks has the wrong shape");
        if (r.mask_of) is(r.mask_of, "mask_of", DType::I32, rows, 0);
    }
}

}  // namespace oxrt
