/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree_f32.hip - the attention of drafted tokens (dsv4_tree.h) over
 * F32 caches. */
#define DSV4_TREE_KERNEL
#include "dsv4_tree.h"

int dsv4_tree_f32_launch(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st)
{
    return tree_format<DSV4_GPU_KV_F32>(a, fmt, kc, (unsigned)(a.ns * a.nb), st);
}
