// The norm of each head of the queries and keys and the rotation by their
// positions in one pass, and its gradients (rotary.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <string>
#include <vector>

#include "branches.hpp"
#include "presk_hip.h"

namespace presk {

// as attn.hpp's: the checks, the workspace, the launches, the spans of a step
std::string rotary_check(const presk_hip_rot& a, int what);
std::string rotary_check_all(const presk_hip_rot& a, int what);
size_t rotary_workspace(const presk_hip_rot& a, int what);
hipError_t rotary_run(const presk_hip_rot& a, int what, hipStream_t s);
void rotary_spans(const presk_hip_rot& a, int what, std::vector<Span>* rd, std::vector<Span>* wr);

}  // namespace presk
