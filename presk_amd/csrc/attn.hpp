// Attention of grouped heads without its weights in memory, and its gradients
// (attn.hip, attn_dev.hpp): softmax(scale q k^T) v over the keys that a query may
// read.
#pragma once

#include <hip/hip_runtime.h>

#include <string>
#include <vector>

#include "branches.hpp"
#include "gemm.hpp"
#include "presk_hip.h"

namespace presk {

// What the ABI's arguments ask for, checked on the host: "" or why not, the
// message starting with its code.  attn_check looks at the type and the sizes,
// attn_check_all at the buffers and the workspace too.
std::string attn_check(const presk_hip_attn& a, int what);
std::string attn_check_all(const presk_hip_attn& a, int what);
// the bytes of workspace a checked call needs
size_t attn_workspace(const presk_hip_attn& a, int what);
// the launches of a checked call
hipError_t attn_run(const presk_hip_attn& a, int what, hipStream_t s);
// the byte spans that a step of a sequence reads and writes
void attn_spans(const presk_hip_attn& a, int what, std::vector<Span>* rd, std::vector<Span>* wr);

// ---- what the kernels share -------------------------------------------------

// element (b, i, h, d) at p + b * batch + i * seq + h * head + d; `vec`: every
// row of d elements is whole 16-byte vectors
struct AttnTensor {
    const void* p;
    long long batch, seq, head;
    int vec;
};

struct AttnArgs {
    AttnTensor q, k, v, o, dout, dq, dk, dv;
    float* lse;                  // [batch][heads][tq], null: not kept
    const long long *lens, *first;
    long long first0;            // where `first` is null
    int batch, heads, kv, per, tq, tk, d;
    int causal, window;          // window 0: none
    int cols;                    // of the mask, 0: none
    // the mask's bits: word w of row i at bits + (b * bits_batch + i) * words + w
    // (bit c of word w is column 32 w + c), and by columns (bit r of word w of
    // column c is row 32 w + r); zero past its ends
    const unsigned *bits, *bits_t;
    int words, words_t;
    long long bits_batch, bits_t_batch;   // rows (columns) from one sequence's to the next one's (0: shared)
    const unsigned char* any;    // [sequences][blocks of 32 rows][words]: whether 32 x 32 of the mask hold any; null: few columns
    float c, scale;              // scale log2 e, scale
    unsigned* flag;
    // the few rows' form: `pack` heads of a group stand beside each other as
    // rows; the keys are cut into `splits`, whose sums are joined after
    int pack, splits, chunk;     // `chunk` keys a split
    float *part, *part_ml;       // [split][batch][heads][tq][ND * 32] and [split][batch][heads][tq]{max, sum}
    // the keys' and values' gradients: `parts` of their rows, summed after
    int parts;                   // (`part`: [dk, dv][part][batch][kv][tk][ND * 32])
    // what the backward pass needs of a row: -lse log2 e and -sum do o
    float* rows;                 // [2][batch][heads][tq]
};

// bits of a byte mask
struct AttnMask {
    const unsigned char* mask;   // element (b, i, c) at mask + b * batch + i * row + c
    long long batch, row;
    int nbatch, tq, cols, words, words_t;
    unsigned *bits, *bits_t;     // bits_t null: not wanted
    unsigned char* any;
};

constexpr int kAttnTile = 128;   // rows of a workgroup
constexpr int kAttnFew = 32;     // rows that are one block of a wave

// nd: 32-wide pieces of a head, 2, 4 or (16-bit) 8
hipError_t attn_fwd_f32(const AttnArgs& a, int nd, hipStream_t s);
hipError_t attn_fwd_bf16(const AttnArgs& a, int nd, hipStream_t s);
hipError_t attn_fwd_f16(const AttnArgs& a, int nd, hipStream_t s);
hipError_t attn_bwd_f32(const AttnArgs& a, int nd, hipStream_t s);
hipError_t attn_bwd_bf16(const AttnArgs& a, int nd, hipStream_t s);
hipError_t attn_bwd_f16(const AttnArgs& a, int nd, hipStream_t s);

}  // namespace presk
