// Paged decode: bf16 queries over a pool of int8.
#include "paged_decode.cuh"

namespace ws {
namespace paged {

int launch_bf16_i8(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    return launch_any<false, true>(a, DB, NT, ctas, st);
}

}  // namespace paged
}  // namespace ws
