// D = 128 instances of the chunk attention kernel with shared prefixes.
#define AKT_CHUNK_TU 128
#define AKT_CHUNK_SHARED
#include "paged_chunk.hip"
