// Where the parts of an expert plan lie (experts.cu writes it, the kernels of experts read it).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/void_b200.h"

namespace vb {

// int32 words: [number of chunks, 0, 0, 0], bounds [experts + 1], chunk_ptr [experts + 1], then (on 16 bytes) chunks [capacity][4]
struct PlanView {
  int32_t *head, *bounds, *chunk_ptr;
  int4* chunks;   // expert, first token, token behind the last, 0
  int capacity;
};
// Every expert's run ends with at most one chunk that is not full, and every chunk holds a token.
inline int64_t plan_capacity(int64_t n_experts, int64_t rows, int64_t chunk) {
  const int64_t most = rows / chunk + n_experts;
  return most < rows ? most : rows;
}
inline int64_t plan_table(int64_t n_experts) { return (4 + 2 * (n_experts + 1) + 3) / 4 * 4; }
inline PlanView plan_of(const void_experts& x, int64_t rows) {
  PlanView v;
  v.head = const_cast<int32_t*>(x.plan);
  v.bounds = v.head + 4;
  v.chunk_ptr = v.bounds + x.n_experts + 1;
  v.chunks = reinterpret_cast<int4*>(v.head + plan_table(x.n_experts));
  v.capacity = (int)plan_capacity(x.n_experts, rows, x.chunk);
  return v;
}

}  // namespace vb
