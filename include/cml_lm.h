/*
 * cml_lm.h -- language models behind one interface: a registry keyed by the architecture a model's own
 * files name, loading, sequences over a paged cache, a step function that runs any mix of prompt portions
 * and decoded tokens as one batch, generation, and the runner of the continuous-batching scheduler
 * (cml_quant_api.h). No C-ML counterpart: C-ML's forward is one LLaMA, one sequence.
 *
 * A model is either a folder with config.json ("architecture" names the class) and model.safetensors, or
 * a GGUF file (class "llama"). Built-in classes: "Rarolorn", "Situlorn", "Lenedra" and
 * "Zevilorn" (folders), "llama" (GGUF).
 *
 * Errors as in cml_quant_api.h: NULL or -1, with a line through cml_log_message.
 */
#ifndef CML_LM_H
#define CML_LM_H

#include <stdint.h>

#include "cml_quant_api.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CMLLanguageModel CMLLanguageModel;

typedef struct CMLLMOptions {
    DType dtype;                /* DTYPE_BFLOAT16: the serving form. DTYPE_FLOAT32: everything in 32-bit */
    int max_tokens;             /* tokens the cache pool holds, all sequences together */
    int max_sequences;          /* sequences open at a time */
    int max_step_rows;          /* tokens of one step; 0: max_tokens */
    int cache;                  /* CML_LM_CACHE_DEFAULT: 16-bit keys and values (32-bit in the 32-bit form). _INT8, _E4M3: 8 bits and a scale for
                                   every 16 tokens and key/value head; serving form of models whose layers all have grouped attention
                                   with heads up to 256, neither convolved nor with mixed scores */
    int weights;                /* CML_LM_WEIGHTS_DEFAULT: as dtype says. _INT8: projections, dense and shared feed-forwards and the vocabulary projection as 8-bit integers with a
                                   scale for each of their rows, multiplied with rows that are brought to 8 bits and a scale each; experts, what makes their router's
                                   logits, and products inside latent attention and recurrences stay bfloat16. Serving form of models from folders */
} CMLLMOptions;
#define CML_LM_WEIGHTS_DEFAULT 0
#define CML_LM_WEIGHTS_INT8 1
#define CML_LM_CACHE_DEFAULT 0
#define CML_LM_CACHE_INT8 1
#define CML_LM_CACHE_E4M3 2

/* One sequence's part of a step: its next tokens, and the places among them (ascending) whose logits are
 * asked for: of all entries together no more than a step may have tokens (or 64, where that is more). */
typedef struct CMLLMEntry {
    int seq;
    const int* tokens;
    int num_tokens;
    const int* want;
    int num_want;
} CMLLMEntry;

CMLLMOptions cml_lm_default_options(void);      /* bfloat16, 8192 tokens, 8 sequences */
int cml_lm_known(const char* architecture);     /* 1: a class of that name is registered */
CMLLanguageModel* cml_lm_load(const char* path, const CMLLMOptions* options);
void cml_lm_free(CMLLanguageModel* lm);
const char* cml_lm_architecture(const CMLLanguageModel* lm);
int cml_lm_vocab_size(const CMLLanguageModel* lm);
CMLTokenizer* cml_lm_tokenizer(const CMLLanguageModel* lm);      /* owned by the model; NULL when it has none */

/* A sequence takes a slot now and cache blocks as it grows; closing it gives both back. */
int cml_lm_sequence_open(CMLLanguageModel* lm);                  /* id, -1: no free slot */
int cml_lm_sequence_close(CMLLanguageModel* lm, int seq);
int cml_lm_sequence_length(CMLLanguageModel* lm, int seq);
/* A new sequence that goes on from where `seq` stands: it shares the blocks that are full, has a copy of the one that is not, and of a recurrence's state.
 * Id, -1: no free slot or block (or a class without a paged pool). */
int cml_lm_sequence_fork(CMLLanguageModel* lm, int seq);
/* The sequence ends after its first `length` tokens. Refused (-1, nothing changes) beyond its end, where keys that the next token will look back to were let go of, inside a block that another
 * sequence shares, and, unless length is what it has, for models that keep a state per sequence. (An 8-bit cache keeps the scales that the dropped tokens asked for.) */
int cml_lm_sequence_truncate(CMLLanguageModel* lm, int seq, int length);
/* Moves the blocks in use to the lowest ids of the pool. Returns how many moved, -1: a call of the device failed, and nothing has changed. */
int cml_lm_compact(CMLLanguageModel* lm);
/* Blocks of the pool (cml_lm_block_size tokens each): all of them, and those not in use. */
int cml_lm_block_size(const CMLLanguageModel* lm);
int cml_lm_blocks_total(const CMLLanguageModel* lm);
int cml_lm_blocks_free(const CMLLanguageModel* lm);

/* Runs all entries as one batch. logits: host fp32 [sum of num_want][vocab], in the order of the entries
 * and of `want`; may be NULL when nothing is wanted. Nothing changes when the arguments are refused (unknown
 * token, a sequence twice, pool or step too small). The "llama" class gives logits of an entry's last token only. */
int cml_lm_step(CMLLanguageModel* lm, const CMLLMEntry* entries, int num_entries, float* logits);
/* The same, but picks the arg-max of every wanted row on the device: picked[sum of num_want]. */
int cml_lm_step_greedy(CMLLanguageModel* lm, const CMLLMEntry* entries, int num_entries, int* picked);
/* The same, but says on the device what the logits of every wanted row mean: the log probability of its token among targets[sum of num_want] (-1: none), the entropy
 * of the row's distribution in nats, and the `top` (0 .. 32) likeliest tokens with their log probabilities, best first, the lower id first among equals
 * (top_ids, top_logprobs [sum of num_want][top]). Outputs that are NULL are left out; targets and logprobs go together. See cmlb200_token_scores. */
int cml_lm_step_scored(CMLLanguageModel* lm, const CMLLMEntry* entries, int num_entries, const int* targets, int top, float* logprobs, float* entropies, int* top_ids,
                       float* top_logprobs);
/* The same, but draws the token of every wanted row on the device, from the softmax of its logits over the row's temperature: temperatures [sum of num_want] (NULL: 1; below 1e-5: the largest
 * logit's token; above 1e30: refused), random [sum of num_want] 64-bit random numbers, each used once (NULL where all temperatures are below 1e-5). picked[sum of num_want], -1 for a row that holds no
 * distribution. Nothing is cut off the distribution. See cmlb200_verify_drafts. */
int cml_lm_step_sampled(CMLLanguageModel* lm, const CMLLMEntry* entries, int num_entries, const float* temperatures, const uint64_t* random, int* picked);
/* Drafted tokens: an entry's first token is the one its sequence goes on with, those behind it are drafts (256 tokens of all entries together; `want` is not looked at). Runs them all, keeps
 * drafts while the model's own distribution would have had them (temperatures and random: one per entry, as above; the drafts count as chosen for certain), and draws the token behind those:
 * accepted[num_entries] drafts kept, next[num_entries] (-1: no distribution). Kept tokens and `next` are distributed as tokens of the model drawn one by one. The sequence then ends behind
 * the kept drafts; `next` is not in it yet. Models that keep a state per sequence take no drafts. An 8-bit cache holds 16 tokens to a scale: there the model's distribution is the one with the drafts of
 * a group in the cache beside the tokens that stay, and where a dropped draft raised the group's scale the kept tokens stay as coarse as it made them. */
int cml_lm_step_verified(CMLLanguageModel* lm, const CMLLMEntry* entries, int num_entries, const float* temperatures, const uint64_t* random, int* accepted, int* next);
/* Greedy decoding that stays on the device: `steps` steps of all sequences, each step's picks the next
 * one's tokens, out_tokens [steps][num_seqs]; *elapsed_ms (optional) is the time of the loop on the device. */
int cml_lm_decode_greedy(CMLLanguageModel* lm, const int* seqs, const int* first_tokens, int num_seqs, int steps, int* out_tokens,
                         float* elapsed_ms);

/* Generates from a prompt through the scheduler: the result holds prompt + generated ids (and the decoded
 * text when the model has a tokenizer). config NULL: greedy, 256 tokens, no end token. */
CMLGenerationResult* cml_lm_generate(CMLLanguageModel* lm, const int* prompt, int num_tokens, const CMLGenerationConfig* config);
/* Generates from a prompt with drafts of another model of the same vocabulary, on the same device: it draws `drafts` (1 .. 32) tokens one by one, of which a step of `lm` keeps what fits its own
 * distribution (cml_lm_step_verified, with the drafter's own probabilities): the result is distributed as cml_lm_step_sampled's, whatever the drafter is, and equals it where config is greedy (up to
 * rounding: a step of several tokens multiplies in other kernels than one of a single token). The same folder loaded with 8-bit weights is a drafter. config NULL: greedy, 256 tokens; its top_k and
 * top_p are not looked at. With an 8-bit cache of `lm` this holds as far as cml_lm_step_verified says. Steps that are shorter than drafts + 1 bring as many drafts as they hold. Neither model may keep a state per sequence, and both hold the prompt and max_new_tokens. stats may be NULL. */
typedef struct CMLLMDraftStats {
    int steps, drafted, accepted;
} CMLLMDraftStats;
CMLGenerationResult* cml_lm_generate_drafted(CMLLanguageModel* lm, CMLLanguageModel* drafter, int drafts, const int* prompt, int num_tokens, const CMLGenerationConfig* config, uint64_t seed,
                                             CMLLMDraftStats* stats);
/* Runs the scheduler over a model until queue and batch are empty or max_steps (> 0) steps were taken: every
 * step is one batch of prompt portions and decoded tokens. A request waits while the pool could not hold it
 * to its end. config gives sampling (NULL: greedy) and the end token; lengths come from the requests.
 * on_finish (optional) sees each request before it is freed. Returns the number of steps, -1 on error. */
int cml_serving_run_lm(CMLServingContext* ctx, CMLLanguageModel* lm, const CMLGenerationConfig* config, int max_steps,
                       void (*on_finish)(const CMLSequenceRequest* request, void* user), void* user);

#ifdef __cplusplus
}
#endif
#endif /* CML_LM_H */
