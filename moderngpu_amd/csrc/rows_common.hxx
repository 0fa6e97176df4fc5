// Argument checks of the row operators (embedding, distillation, sampling).
#pragma once
#include "launcher_common.hxx"
#include <moderngpu/rows.hxx>

namespace mgpu_hip {

inline size_t row_value_size(int dtype) {
  switch(dtype) {
    case MGPU_F32: return 4;
    case MGPU_F16: case MGPU_BF16: return 2;
  }
  return 0;
}

// Calls f with a null pointer of dtype's value type.
template<typename f_t>
int with_row_type(int dtype, f_t f) {
  switch(dtype) {
    case MGPU_F32: return f((float*)nullptr);
    case MGPU_F16: return f((mgpu::f16_t*)nullptr);
    case MGPU_BF16: return f((mgpu::bf16_t*)nullptr);
  }
  return (int)hipErrorInvalidValue;
}

// A matrix argument: where it lies in memory.
struct matrix_t {
  const char* begin;
  int64_t rows, cols, stride;
  size_t value;

  matrix_t(const void* p, int64_t rows, int64_t cols, int64_t stride,
    size_t value) : begin((const char*)p), rows(rows), cols(cols),
    stride(stride), value(value) { }

  bool empty() const { return rows <= 0 || cols <= 0; }
  // Pointer there and aligned to a value, stride in range, and every byte
  // offset fits 63 bits.
  bool input_ok() const {
    if(empty()) return true;
    return begin && 0 == (uintptr_t)begin % value && stride >= 0 &&
      stride <= ((int64_t)1 << 62) / (int64_t)value / rows - cols;
  }
  bool output_ok() const {
    return input_ok() && (empty() || rows == 1 || stride >= cols);
  }
  const char* end() const {
    return begin + value * ((rows - 1) * stride + cols);
  }
  bool overlaps(const matrix_t& other) const {
    return !empty() && !other.empty() && begin < other.end() &&
      other.begin < end();
  }
};

} // namespace mgpu_hip
