// kr_kv_attend_8.hip -- attention over the paged cache, eight bits (a file for each width: they compile side by side).
#include "kr_kv_step_dev.h"
#include "kr_kv_tile_dev.h"

int kr_launch_kv_step_8(const KvAttnArgs& a, int dim, int half, hipStream_t st) { return kvs_dim<1>(a, dim, half, st); }
int kr_launch_kv_tile_8(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st) { return kvt_dim<1>(a, dim, half, waves, st); }
