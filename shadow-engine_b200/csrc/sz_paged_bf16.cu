// The attention kernels over a paged cache of this element type (one file a type, so that they compile side by side).
#include "sz_paged.cuh"

PgKernels pg_kernels_bf16(bool wide, int hd, int nqt) { return pg_of<PG_BF16>(wide, hd, nqt); }
