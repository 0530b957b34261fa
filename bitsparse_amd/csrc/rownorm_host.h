// Host-side pieces that the forward and backward entry points of the step
// between two blocks share.
#pragma once

#include "bs_host.h"
#include "philox.h"
#include "rownorm.h"

namespace bs {

// BS_ERR_INVALID with a message for arguments that no kernel takes
int join_check(const bs_join* args, const char* what);

// the rule of a dropout, and whether a step takes it
int drop_rule(const bs_drop* d, const char* what, DropRule* r);
int join_drop_check(const bs_join& j, const bs_drop* drop, const char* what, DropRule* r);

RowParam row_param(const bs_vector& v, int per);

}  // namespace bs
