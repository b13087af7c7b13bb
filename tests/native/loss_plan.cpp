// The graph-branch planner (presk_amd/csrc/branches.hpp) over steps that are
// losses, by the spans that a recorded sequence gives it of one
// (presk_amd/csrc/loss_buffers.hpp); built and read by tests/test_loss_plan.py.
// Input (the file named by argv[1]), a step a line:
//   L <head> <what> <type> <rows> <model> <vocab> <top> <x> <w> <index>
//     <teacher> <loss> <lse> <mean> <ct> <dx> <dw> <flag> <work> <work bytes>
//   C <src> <dst> <flag> <from> <to> <n>        an edge conversion
// Output, for argv[2] branches, a step a line: its stream, then the steps it
// waits for.
#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <string>
#include <vector>

#include "loss_buffers.hpp"

using namespace presk;

int main(int argc, char** argv) {
    if (argc < 3) return 2;
    std::ifstream in(argv[1]);
    std::vector<BranchStep> steps;
    std::string tag;
    auto ptr = [&]() {
        unsigned long long v = 0;
        in >> v;
        return (void*)(uintptr_t)v;
    };
    while (in >> tag) {
        BranchStep st;
        if (tag == "L") {
            presk_hip_loss a{};
            bool head;
            int what;
            std::string type;
            in >> head >> what >> type >> a.rows >> a.model >> a.vocab >> a.top;
            a.dtype = type.c_str();
            a.x = ptr();
            a.w = ptr();
            a.index = (const int64_t*)ptr();
            a.teacher = ptr();
            a.loss = (float*)ptr();
            a.lse = (float*)ptr();
            a.mean = (float*)ptr();
            a.ct = (const float*)ptr();
            a.dx = ptr();
            a.dw = ptr();
            a.flag = (uint32_t*)ptr();
            a.work = ptr();
            in >> a.work_bytes;
            loss_spans(a, what, head, &st.rd, &st.wr);
        } else if (tag == "C") {
            void* const src = ptr();
            void* const dst = ptr();
            void* const flag = ptr();
            st.bufs = {src, dst, flag};
            in >> st.from >> st.to >> st.n;
        } else {
            return 3;
        }
        if (!in) return 4;
        steps.push_back(std::move(st));
    }
    std::vector<int> lane;
    std::vector<std::vector<std::pair<int, int>>> waits;
    plan_branches(steps, std::atoi(argv[2]), &lane, &waits);
    for (size_t i = 0; i < steps.size(); ++i) {
        std::printf("%d", lane[i]);
        for (const auto& w : waits[i]) std::printf(" %d", w.second);
        std::printf("\n");
    }
    return 0;
}
