/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree_bf16.hip - the attention of drafted tokens (dsv4_tree.h) over
 * BF16 caches. */
#define DSV4_TREE_KERNEL
#include "dsv4_tree.h"

int dsv4_tree_bf16_launch(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st)
{
    return tree_format<DSV4_GPU_KV_BF16>(a, fmt, kc, (unsigned)(a.ns * a.nb), st);
}
