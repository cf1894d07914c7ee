// Paged decode: fp16 queries over a pool of the same type.
#include "paged_decode.cuh"

namespace ws {
namespace paged {

int launch_f16(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    return launch_any<true, false>(a, DB, NT, ctas, st);
}

}  // namespace paged
}  // namespace ws
