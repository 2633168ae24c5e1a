// Launchers of the embedding lookup and its gradient by sorted tokens (embed.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace oxi {
// out[t] = w[ids[t]] * scale ([T, H]; bf16 or f32 with w).  An id outside [0, V) gives a zero row and
// records a bounds error in the status word.
void launch_embedding_fwd(const int64_t* ids, const void* w, void* out, bool bf16, int64_t T, int64_t V, int H,
                          float scale, int* status, cudaStream_t st);

// Workspace of the gradient, in bytes.
int64_t embedding_bwd_workspace(int64_t T, int H);
// dw[v] = scale * sum over the tokens t with ids[t] == v of dy[t], summed in f32 in the order of t.
//   accumulate: dw is f32 [V, H] and is added to (rows that no token names stay as they are)
//   otherwise:  dw has dy's type, and every row is written
void launch_embedding_bwd(const int64_t* ids, const void* dy, bool bf16, void* dw, bool accumulate, int64_t T,
                          int64_t V, int H, float scale, void* workspace, cudaStream_t st);
}  // namespace oxi
