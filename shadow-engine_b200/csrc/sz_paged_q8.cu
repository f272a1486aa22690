// The attention kernels over a paged cache of this element type (one file a type, so that they compile side by side).
#include "sz_paged.cuh"

PgKernels pg_kernels_q8(bool wide, int hd, int nqt) { return pg_of<PG_Q8>(wide, hd, nqt); }
