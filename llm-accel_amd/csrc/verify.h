// verify.h -- next-token probabilities and draft verification over the LM
// head's scores (internal to the library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llm {

// Scores per workgroup of the passes over a row, and the most such chunks.
constexpr uint32_t kProbChunk = 2048;
constexpr uint32_t kProbChunksMax = 128;  // vocab < 2^18
// Entries of one of the two tables of powers of two.
constexpr uint32_t kExp2Entries = 1024;

struct ProbArgs {
    const int64_t* scores;  // [rows][lds], 20 fraction bits
    uint32_t lds, vocab, rows;
    const uint32_t* exp2;   // [2][kExp2Entries]: 2^-(i / 2^10), 2^-(i / 2^20) in 2^-30
    uint32_t inverse[8];    // per row log2(e) / temperature in 2^-24
    unsigned long long* keys;  // the rows' argmax keys; 0 once the call's work is done
    // per row the largest score, per row and chunk the sum of its weights
    int64_t* top;              // [8]
    unsigned long long* part;  // [8][kProbChunksMax]
};
// Q0.32 probabilities probs[r][v], tight rows.
hipError_t launch_probs(const ProbArgs& a, uint32_t* probs, hipStream_t st);

struct VerifyArgs {
    ProbArgs p;
    uint32_t requests;
    uint32_t first[8], count[8];  // per request its first row and its drafts
    uint32_t draft0[8];           // its first row of `q`
    uint32_t draft[8];            // per row its drafted token (a request's last row: unused)
    uint32_t accept_u[8];         // per row
    uint32_t sample_u[8];         // per request
    const uint32_t* q;            // [drafts][vocab] Q0.32, or null: all on the drafted token
    // per request and chunk the sums of what a token is drawn from (the part
    // above q, and p itself), arrival counters (one line per request, then
    // one of the whole; zero between launches)
    unsigned long long* left;     // [8][kProbChunksMax][2]
    uint32_t* count_in;           // [9 * 32]
    // pinned host memory: accepted[8], token[8], prob[8 rows], and the word
    // that receives seq once they are visible
    uint32_t* host;
    uint32_t* flag;
    uint32_t seq;
};
hipError_t launch_verify(const VerifyArgs& a, hipStream_t st);

}  // namespace llm
