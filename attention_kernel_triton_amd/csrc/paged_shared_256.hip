// D = 256 instances of the chunk attention kernel with shared prefixes.
#define AKT_CHUNK_TU 256
#define AKT_CHUNK_SHARED
#include "paged_chunk.hip"
