// Host entry points of the kernels for few query rows on a shared prefix and own keys, compiled once per 16-bit element type
// (na2d_prefix_tc.cu with -DNA2D_TC_DT=1 for bf16 and 2 for fp16).
#pragma once

#include "na2d_attn.cuh"

namespace na2d_prefix {

constexpr int kTokenEntries = 4096;     // prefixes and batch entries on the line, at most
// Steps that a unit counts for beside those of its keys: its queries' way in and its sums' way out.  64 x 8 caches of 1 to 1024 keys behind a prefix of
// 16384: 73.1 us with 1, 70.8 with 3, 71.3 with 6; 16 x 4 prefixes of up to 8192 with 256 short caches 48.7, 47.6, 47.6, of up to 32768 130.0,
// 130.1, 136.0.
constexpr int kUnitSteps = 3;

// One kind of keys: prefixes, or the entries' own.
struct TokenSide {
    na2d_attn::Operand k, v;            // (entries, Nk, T, C)
    const int* lengths;
    int entries, T;                     // entries 0: this side is not on the line
    int share;                          // batch entries of one
    int rows;                           // of a unit: G share Tq, row (h share + a) Tq + t
    size_t first_row;                   // of its parts in the workspace
};
struct Tokens {
    TokenSide side[2];                  // prefixes, own
    na2d_attn::Operand q;               // (B, N, Tq, C)
    int N, Nk, G, Tq, C, causal;
    int least;                          // steps of 16 keys that a warp takes, at least
    int behind;                         // another kernel of the call has been launched before
    float sl2;
    na2d_attn::Div by_tq, by_n, by_g;
    int* table;                         // steps before each entry, of all, and those of a warp
    float *part_o, *part_lse;
};
// Where a row's sums over the prefix come from: the line (count 0), or another kernel's results, (count, entries, N, share Tq).  (Own keys are
// on the line in every call that has one.)
struct JoinPrefix {
    const float *o, *lse;
    size_t stride;                      // rows from one to the next
    int count, share;
    na2d_attn::Div by_share;
};

// Query rows of a unit that the kernel takes, at most.
constexpr int kTokenRows = 32;
// Warps of the line.
inline int token_warps(int sms) { return sms * 8; }

int tokens_bf16(const na2d_attn::Place& at, const Tokens& x, const JoinPrefix& prefix, void* o, float* lse, int B);
int tokens_f16(const na2d_attn::Place& at, const Tokens& x, const JoinPrefix& prefix, void* o, float* lse, int B);

}  // namespace na2d_prefix
