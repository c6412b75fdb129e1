// kve.h -- the evicting KV cache's layout, shared by its write side (kve_append.hip), its
// attention (kve_decode.hip) and its eviction (kve_evict.hip).
//
// Token slot t of a sequence lies in slot t % P of page block_table[sequence][t / P]; a page
// holds, for each kv head, P rows of D values of keys and of values, P weights (fp32: the
// softmax weights that the token got so far) and P positions (int32).  A row of the pool is
// (page * Hkv + head) * P + slot.
#pragma once

#include "kv4.h"

namespace ojx {

struct KveView {
    char *k, *v;                // rows of D values
    float *w;
    int *pos;
    const int *bt;              // [B][max_pages]
    const double *turns;        // [rot / 2] or null
    int B, max_pages, pshift, num_pages;   // page = 1 << pshift slots
    int Hkv, D, dtype, rot, interleaved;
    int cap;                    // slots of a sequence: max_pages pages
};

int kve_view(const OjasxKVECache *c, KveView *v);   // 0 or an error code

// The pool row of sequence b's slot t (0 <= t < cap) and kv head 0, or -1 where the block
// table maps no page of the pool; kv head h's is h << pshift rows further.
__device__ __forceinline__ long kve_row(const KveView &c, int b, int t) {
    const int page = c.bt[(long)b * c.max_pages + (t >> c.pshift)];
    if (page < 0 || page >= c.num_pages) return -1;
    return (((long)page * c.Hkv) << c.pshift) + (t & ((1 << c.pshift) - 1));
}

}  // namespace ojx
