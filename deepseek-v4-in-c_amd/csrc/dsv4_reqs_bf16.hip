/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_reqs_bf16.hip - the attention of a batch's requests (dsv4_tree.h) over
 * BF16 caches. */
#define DSV4_TREE_KERNEL
#include "dsv4_tree.h"

int dsv4_reqs_bf16_launch(const Dsv4ReqsJob &a, int fmt, int kc, unsigned groups, hipStream_t st)
{
    return tree_format<DSV4_GPU_KV_BF16>(a, fmt, kc, groups, st);
}
