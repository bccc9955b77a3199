// D = 64 instances of the chunk attention kernel.
#define AKT_CHUNK_TU 64
#include "paged_chunk.hip"
