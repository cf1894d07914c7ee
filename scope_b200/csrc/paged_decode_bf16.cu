// Paged decode: bf16 queries over a pool of bf16.
#include "paged_decode.cuh"

namespace ws {
namespace paged {

int launch_bf16(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    return launch_any<false, k16, false>(a, DB, NT, ctas, st);
}

}  // namespace paged
}  // namespace ws
