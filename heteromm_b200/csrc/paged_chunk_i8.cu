// paged_chunk_i8.cu — the chunk kernel over a cache held in int8 codes.
#include "paged_chunk.cuh"

namespace hmm {
namespace serve {

template hmm_status_t run_chunk<CODEC_I8>(const AttnArgs&, bool, int, bool, unsigned char*, cudaStream_t, ChunkJoin*);

}  // namespace serve
}  // namespace hmm
