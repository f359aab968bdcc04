// Shared by the paged cache's kernels.
#pragma once
#include "kq_attn.h"

// The pool's pointers, shape, strides and alignment (a kq_status).
int kq_pool_check(const kq_paged_pool *pool);
