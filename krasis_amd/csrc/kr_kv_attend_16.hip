// kr_kv_attend_16.hip -- attention over the paged cache, 16-bit pages (a file for each width: they compile side by side).
#include "kr_kv_step_dev.h"
#include "kr_kv_tile_dev.h"

int kr_launch_kv_step_16(const KvAttnArgs& a, int dim, int half, hipStream_t st) { return kvs_dim<0>(a, dim, half, st); }
int kr_launch_kv_tile_16(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st) { return kvt_dim<0>(a, dim, half, waves, st); }
