// verify.h -- next-token probabilities and draft verification over the LM
// head's scores (internal to the library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llm {

// Scores per workgroup of the passes over a row, and the most such chunks: the
// sums' arrivals and the draws' share a line each, and arrivals on one line
// serialise (1,192 of them, 1,024 scores each, on one: the pass took 22 us; in
// chunks of 4,096 and a line per row 10).
constexpr uint32_t kSumChunk = 4096, kSumChunksMax = 64;  // vocab < 2^18
constexpr uint32_t kProbChunk = 2048, kProbChunksMax = 128;
// Entries of one of the two tables of powers of two.
constexpr uint32_t kExp2Entries = 1024;

// Where a request's token is drawn: its row, that row's sum of weights and
// largest score, and P of each of its drafts.
struct DrawPlace {
    unsigned long long total;
    int64_t top;
    uint32_t at;  // drafts taken: the request's row of that number
    uint32_t pdraft[7];
};

struct ProbArgs {
    const int64_t* scores;  // score_at(token, row, rows), 20 fraction bits
    uint32_t vocab, rows;
    const uint32_t* exp2;   // [2][kExp2Entries]: 2^-(i / 2^10), 2^-(i / 2^20) in 2^-30
    uint32_t inverse[8];    // per row log2(e) / temperature in 2^-24
    unsigned long long* keys;  // the rows' argmax keys; 0 once the call's work is done
    // requests: per row the one it belongs to; per request its first row, its
    // drafts, its first row of `q`, and 32-bit uniform numbers
    uint32_t requests;
    uint32_t request[8], first[8], count[8], draft0[8], sample_u[8];
    uint32_t draft[8], accept_u[8];  // per row (a request's last: unused)
    const uint32_t* q;      // [drafts][vocab] Q0.32, or null: all on the drafted token
    // per row and chunk the sum of its weights, per request what comes of them
    unsigned long long* part;  // [8][kSumChunksMax]
    DrawPlace* place;          // [8]
    uint32_t* count_in;        // [16 * 32] arrivals, a line per row and per request
                               // (zero between launches)
    // per request and chunk the sums of what a token is drawn from (the part
    // above q, and p itself)
    unsigned long long* left;  // [8][kProbChunksMax][2]
    // pinned host memory: accepted[8], token[8], prob[8 rows], each with seq in
    // its upper half (no word waits for another)
    unsigned long long* host;
    uint32_t seq;
};
// Q0.32 probabilities probs[r][v], tight rows: every row a request without
// drafts.
hipError_t launch_probs(const ProbArgs& a, uint32_t* probs, hipStream_t st);
hipError_t launch_verify(const ProbArgs& a, hipStream_t st);

}  // namespace llm
