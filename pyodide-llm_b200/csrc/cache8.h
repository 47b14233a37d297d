// cache8.h — what the entries of the paged 8-bit cache share.
#pragma once

namespace b200 {

// the pool's arguments as every entry checks them (message under the entry's name); 0 or B200FWD_EINVAL
int check_cache8(const char *what, const void *kc, const void *ks, const void *vc, const void *vs, int blocks,
                 int block, int nkv, int hs);

}  // namespace b200
