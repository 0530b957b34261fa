// Host-side pieces that the forward and backward entry points of the step
// between two blocks share.
#pragma once

#include "bs_host.h"
#include "rownorm.h"

namespace bs {

// BS_ERR_INVALID with a message for arguments that no kernel takes
int join_check(const bs_join* args, const char* what);

RowParam row_param(const bs_vector& v, int per);

}  // namespace bs
