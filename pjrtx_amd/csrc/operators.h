// Custom-call targets of a decoder's serving and training step: attention and
// row writes over a paged key-value cache, the residual norm, and token log
// probabilities, with the gradients of the last two (operators.cc).
#pragma once

#include <map>
#include <string>
#include <vector>

#include "ir.h"
#include "planner.h"
#include "runtime.h"

namespace pjrtx {

// Turns a custom call of one of the targets into its op after checking its
// operands, results and configuration (INVALID_ARGUMENT, or UNIMPLEMENTED for
// sizes outside what the kernels take). False for another target.
bool lower_operator_call(const Program& prog, Op* op);

// The ops' library kinds; kCopy for another op.
LibKind operator_lib_kind(OpKind k);

// Bytes that an operator's step moves at most: its operands and results, but of
// a cache's pages the rows that it writes, or those that its page table names.
double operator_bytes(const Program& prog, const Step& step);

// Runs an operator's step: its results are allocated, or, where the step
// writes operand k in place, result k is operand k's buffer.
void run_operator(Device* dev, const Program& prog, const Step& step, std::vector<MemRef>& vals);

}  // namespace pjrtx
