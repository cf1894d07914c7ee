// Paged differential attention: fp16 queries over a pool of e4m3.
#include "paged_decode.cuh"

namespace ws {
namespace paged {

int launch_diff_f16_e4(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    return launch_any<true, kE4M3, true>(a, DB, NT, ctas, st);
}

}  // namespace paged
}  // namespace ws
