// Launchers of the embedding lookup and its gradient by sorted tokens (embed.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace oxi {
// out[t] = w[ids[t]] * scale ([T, H]; bf16 or f32 with w).  An id outside [0, V) gives a zero row and
// records a bounds error in the status word.  order (null, or embedding_order_bytes(T, V), and scratch as much again):
// the tokens in the order of their ids, for the gradient; it is made beside the lookup.
void launch_embedding_fwd(const int64_t* ids, const void* w, void* out, bool bf16, int64_t T, int64_t V, int H,
                          float scale, int* status, void* order, void* scratch, cudaStream_t st);
// 0: the gradient needs no order (few tokens), or refuses the sizes
int64_t embedding_order_bytes(int64_t T, int64_t V);

// Workspace of the gradient, in bytes (ordered: an order is at hand).
int64_t embedding_bwd_workspace(int64_t T, int H, bool ordered);
// dw[v] = scale * sum over the tokens t with ids[t] == v of dy[t], summed in f32 in an order that T alone decides:
// that of t, in stretches.  order: of the same ids and V, or null.
//   accumulate: dw is f32 [V, H] and is added to (rows that no token names stay as they are)
//   otherwise:  dw has dy's type, and every row is written
void launch_embedding_bwd(const int64_t* ids, const void* order, const void* dy, bool bf16, void* dw, bool accumulate,
                          int64_t T, int64_t V, int H, float scale, void* workspace, cudaStream_t st);
}  // namespace oxi
