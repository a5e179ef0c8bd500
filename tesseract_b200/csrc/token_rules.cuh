// What a request's rules make of a logit (token_rules.cu writes it out, token_choice.cu chooses from it).
//
//   x = l;  x = x / r if x > 0 else x * r      r: repetition, for tokens of the prompt or the answer
//   x = x - f c;  x = x - p if c > 0           f: frequency, p: presence, c: times that the answer has the token
//   x = x + b;  -inf where the mask does not allow the token
//
// in 64 bits, every operation rounded as it stands and the result once to 32 bits: a token that no rule touches keeps its logit's bits,
// and both kernels make the same number of the others.  (Few tokens are touched, so 64 bits cost nothing that shows.)
#pragma once

#include "common.cuh"

enum RuleKind : int { kPenalties = 1, kBiases = 2, kMask = 4 };

constexpr int kMaxBiases = 1024;

// One slot's row of the table (32 bytes).
struct SlotRules {
    int kinds, biases;                   // which rules the slot has; how many entries its list of biases has
    float repetition, presence, frequency;
    int pad[3];
};

struct Rules {
    const int* slots;                    // [rows]: a row's slot, or -1 (no rules); null: no row has rules
    const SlotRules* table;              // [slots]
    const uint32_t* seen;                // [slots][words]: a bit a token of the prompt or the answer
    const int* counts;                   // [slots][stride]: times that the answer has the token
    const uint32_t* masks;               // [slots][words]: a bit a token that may come next
    const int* bias_ids;                 // [slots][room], no id twice; ids outside the vocabulary name nothing
    const float* biases;
    int slot_count, words, stride, room;
};

__device__ __noinline__ float shaped_logit(float l, const SlotRules& rule, bool seen, int count, float bias) {
    double x = (double)l;
    if (seen) x = x > 0.0 ? __ddiv_rn(x, (double)rule.repetition) : __dmul_rn(x, (double)rule.repetition);
    if (count != 0) x = __dsub_rn(x, __dmul_rn((double)rule.frequency, (double)count));
    if (count > 0) x = __dsub_rn(x, (double)rule.presence);
    return __double2float_rn(__dadd_rn(x, (double)bias));
}
