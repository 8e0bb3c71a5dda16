// Which memory an operator may write, seen from what it reads: checks of
// addresses and strides on the host, shared by the library and the module
// that calls it.
#pragma once

#include <cstdint>

#include "../../include/cresso_hip.h"

namespace cresso {

// `rows` rows of `bytes` bytes at a stride of `stride` bytes.
struct RowSpan {
    const void* at;
    int64_t rows, bytes, stride;
};
inline bool empty(const RowSpan& s) { return !s.at || s.rows < 1 || s.bytes < 1; }

// Whether a byte of one may be a byte of the other.  Rows at one common stride
// may lie side by side (slices of one buffer's columns); at different strides
// whatever lies between the first byte and the last counts.
inline bool overlap(const RowSpan& a, const RowSpan& b) {
    if (empty(a) || empty(b)) return false;
    const uintptr_t a0 = (uintptr_t)a.at, b0 = (uintptr_t)b.at;
    const uintptr_t a1 = a0 + (uintptr_t)((a.rows - 1) * a.stride + a.bytes), b1 = b0 + (uintptr_t)((b.rows - 1) * b.stride + b.bytes);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.stride != b.stride || a.stride < 1) return true;
    const int64_t s = a.stride, off = (((int64_t)(b0 - a0)) % s + s) % s;   // where b's rows begin between two of a's
    return off < a.bytes || off + b.bytes > s;
}

// What `grad` shares memory with among a descriptor's inputs, other than the
// logits at the same address and stride, or NULL.  Sizes and types are checked.
inline const char* distill_overlap(const cresso_distill_desc& d) {
    const auto bytes = [](int32_t code) -> int64_t { return code == CRESSO_F32 ? 4 : 2; };
    const int64_t size = bytes(d.dtype), tsize = bytes(d.teacher_dtype);
    const RowSpan grad{d.grad, d.rows, d.vocab * size, d.grad_stride * size};
    const RowSpan logits{d.logits, d.rows, d.vocab * size, d.logits_stride * size};
    const bool in_place = d.grad == d.logits && (d.rows < 2 || d.grad_stride == d.logits_stride);
    if (!in_place && overlap(grad, logits)) return "logits";
    if (overlap(grad, {d.index, d.rows, (int64_t)d.top * d.index_bytes, d.index_stride * d.index_bytes})) return "teacher's indexes";
    if (overlap(grad, {d.teacher, d.rows, d.top * tsize, d.teacher_stride * tsize})) return "teacher's logits";
    if (d.labels && overlap(grad, {d.labels, 1, d.rows * d.label_bytes, 0})) return "labels";
    if (overlap(grad, {d.weights, 1, d.rows * 4, 0})) return "row weights";
    if (overlap(grad, {d.d_loss, d.d_loss ? d.rows : 0, 4, d.d_loss_stride * 4})) return "gradient that arrives";
    if (overlap(grad, {d.stats, d.stats ? 1 : 0, d.rows * 12, 0})) return "stats";
    return nullptr;
}

}  // namespace cresso
