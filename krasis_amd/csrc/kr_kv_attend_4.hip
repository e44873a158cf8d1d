// kr_kv_attend_4.hip -- attention over the paged cache, four bits (a file for each width: they compile side by side).
#include "kr_kv_step_dev.h"
#include "kr_kv_tile_dev.h"

int kr_launch_kv_step_4(const KvAttnArgs& a, int dim, int half, hipStream_t st) { return kvs_dim<2>(a, dim, half, st); }
int kr_launch_kv_tile_4(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st) { return kvt_dim<2>(a, dim, half, waves, st); }
