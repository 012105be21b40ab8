// paged_chunk_e4m3.cu — the chunk kernel over a cache held in e4m3 codes.
#include "paged_chunk.cuh"

namespace hmm {
namespace serve {

template hmm_status_t run_chunk<CODEC_E4M3>(const AttnArgs&, bool, int, bool, unsigned char*, cudaStream_t, ChunkJoin*);

}  // namespace serve
}  // namespace hmm
