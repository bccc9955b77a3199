// D = 256 instances of the chunk attention kernel.
#define AKT_CHUNK_TU 256
#include "paged_chunk.hip"
