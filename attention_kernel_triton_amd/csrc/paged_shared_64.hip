// D = 64 instances of the chunk attention kernel with shared prefixes.
#define AKT_CHUNK_TU 64
#define AKT_CHUNK_SHARED
#include "paged_chunk.hip"
