// The key-value cache in 8 bits: the kernels of kv_cache.h and kv_attend.h for pages of e4m3 numbers, behind the C-ABI of bam_kv.hip.
#include "kv_attend.h"

void kv8_rows(const bam_kv_t* kv, const kv_seqs& s, const kv_rows& io, const bool write, hipStream_t st)
{
    if (write) launch_rows<1, true>(kv, s, io, st);
    else launch_rows<1, false>(kv, s, io, st);
}

void kv8_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st)
{
    if (kv->f16) launch_attend<1, 1>(kv, s, a, p, st);
    else launch_attend<0, 1>(kv, s, a, p, st);
}
