/* Generation with a drafter (cml_lm.h): another model draws tokens one by one, and one step of the model itself keeps those that fit its own distribution. */
#include <stdlib.h>
#include <string.h>
#include <time.h>

#include "cml_lm_internal.h"

#define MOST_DRAFTS 32

/* A sequence of 64-bit random numbers (Steele, Lea, Flood: Fast splittable pseudorandom number generators, 2014): every drawn token gets one of its own. */
static uint64_t next_random(uint64_t* state) {
    uint64_t z = *state += 0x9E3779B97F4A7C15u;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9u;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBu;
    return z ^ (z >> 31);
}

typedef struct Drafting {
    CMLLanguageModel *lm, *drafter;
    int seq, draft_seq;            /* -1: not open */
    float temperature;
    uint64_t random;
    float* d_probabilities;        /* the drafter's logits of this round's drafts */
    size_t row;                    /* bytes */
} Drafting;

/* Tokens into a model, as many tokens as a step takes at a time; picked: the token drawn behind it (NULL: none). */
static int read_prompt(Drafting* d, CMLLanguageModel* lm, int seq, int portion, const int* tokens, int n, int* picked) {
    for (int at = 0; at < n; at += portion) {
        const int k = n - at < portion ? n - at : portion, last = k - 1, ask = picked && at + k == n;
        const CMLLMEntry e = {seq, tokens + at, k, &last, ask};
        const uint64_t r = ask ? next_random(&d->random) : 0;
        if (ask ? cml_lm_step_sampled(lm, &e, 1, &d->temperature, &r, picked) : cml_lm_step(lm, &e, 1, NULL)) return -1;
    }
    return 0;
}

/* Draws `count` drafts behind all n tokens, of which the drafter's sequence holds fewer. */
static int draw_drafts(Drafting* d, const int* tokens, int n, int count, int* drafts) {
    const int has = cml_lm_sequence_length(d->drafter, d->draft_seq);
    for (int i = 0; i < count; i++) {
        if (read_prompt(d, d->drafter, d->draft_seq, cml_lm_step_rows(d->drafter), i ? drafts + i - 1 : tokens + has, i ? 1 : n - has, drafts + i)) return -1;
        if (drafts[i] < 0) return i;                       /* (no distribution: the drafts end here) */
        if (CML_DEV_FAIL(cmlb200_memcpy_d2d((char*)d->d_probabilities + (size_t)i * d->row, cml_lm_logits(d->drafter), d->row, NULL), __func__) || CML_DEV_FAIL(cmlb200_stream_sync(NULL), __func__))
            return -1;
    }
    return count;
}

CMLGenerationResult* cml_lm_generate_drafted(CMLLanguageModel* lm, CMLLanguageModel* drafter, int drafts, const int* prompt, int num_tokens, const CMLGenerationConfig* config, uint64_t seed,
                                             CMLLMDraftStats* stats) {
    static const char* who = "cml_lm_generate_drafted";
    if (!lm || !drafter || lm == drafter || !prompt || num_tokens <= 0 || drafts < 1 || drafts > MOST_DRAFTS) { LOG_ERROR("%s: invalid arguments (up to %d drafts)", who, MOST_DRAFTS); return NULL; }
    if (!cml_lm_takes_drafts(lm) || !cml_lm_takes_drafts(drafter)) { LOG_ERROR("%s: a model keeps no paged cache, or a state per sequence", who); return NULL; }
    if (cml_lm_vocab_size(lm) != cml_lm_vocab_size(drafter)) { LOG_ERROR("%s: vocabularies of %d and %d tokens", who, cml_lm_vocab_size(lm), cml_lm_vocab_size(drafter)); return NULL; }
    CMLGenerationConfig c = cml_generation_default_config();
    c.do_sample = false;
    c.eos_token_id = -1;
    if (config) c = *config;
    if (c.max_new_tokens <= 0) c.max_new_tokens = 256;
    if ((long)num_tokens + c.max_new_tokens > cml_lm_longest(lm) || (long)num_tokens + c.max_new_tokens > cml_lm_longest(drafter)) {
        LOG_ERROR("%s: %d tokens behind %d, sequences of %ld and %ld", who, c.max_new_tokens, num_tokens, cml_lm_longest(lm), cml_lm_longest(drafter));
        return NULL;
    }
    if (drafts > cml_lm_step_rows(lm) - 1) drafts = cml_lm_step_rows(lm) - 1;
    Drafting d = {lm, drafter, -1, -1, c.do_sample ? c.temperature : 0.0f, seed, NULL, (size_t)cml_lm_vocab_size(lm) * sizeof(float)};
    CMLLMDraftStats s = {0, 0, 0};
    struct timespec t0, t1;
    clock_gettime(CLOCK_MONOTONIC, &t0);
    CMLGenerationResult* res = (CMLGenerationResult*)calloc(1, sizeof *res);
    int ok = res && (res->token_ids = (int*)malloc((size_t)(num_tokens + c.max_new_tokens + MOST_DRAFTS + 1) * sizeof(int))) != NULL;
    const int end = num_tokens + c.max_new_tokens;
    int n = num_tokens, token = -1, done = 0;
    if (ok) memcpy(res->token_ids, prompt, (size_t)num_tokens * sizeof(int));
    /* what a rejected draft took may be behind a window by then */
    cml_lm_keep_behind(drafter, drafts + 1);
    ok = ok && !CML_DEV_FAIL(cmlb200_malloc((void**)&d.d_probabilities, (size_t)(drafts + 1) * d.row), who) && (d.seq = cml_lm_sequence_open(lm)) >= 0 && (d.draft_seq = cml_lm_sequence_open(drafter)) >= 0 &&
         !read_prompt(&d, lm, d.seq, cml_lm_step_rows(lm), prompt, num_tokens, &token) && !read_prompt(&d, drafter, d.draft_seq, cml_lm_step_rows(drafter), prompt, num_tokens, NULL);
    if (ok && token < 0) { LOG_ERROR("%s: the prompt's logits hold no distribution", who); ok = 0; }
    if (ok) {
        res->token_ids[n++] = token;
        done = token == c.eos_token_id;
    }
    while (ok && !done && n < end) {
        int run[MOST_DRAFTS + 1], kept, next;
        const int want = end - n - 1 < drafts ? end - n - 1 : drafts, got = want ? draw_drafts(&d, res->token_ids, n, want, run + 1) : 0;
        if (got < 0) { ok = 0; break; }
        run[0] = res->token_ids[n - 1];
        const CMLLMEntry e = {d.seq, run, got + 1, NULL, 0};
        const uint64_t r = next_random(&d.random);
        if (cml_lm_run_verified(lm, &e, 1, &d.temperature, &r, d.d_probabilities, &kept, &next, who)) { ok = 0; break; }
        if (next < 0) { LOG_ERROR("%s: a row of logits holds no distribution", who); ok = 0; break; }
        s.steps++;
        s.drafted += got;
        s.accepted += kept;
        for (int i = 0; i <= kept && !done && n < end; i++) {
            res->token_ids[n] = i < kept ? run[1 + i] : next;
            done = res->token_ids[n++] == c.eos_token_id;
        }
        /* the drafter's sequence: what it was fed of the tokens that stay */
        const int fed = cml_lm_sequence_length(drafter, d.draft_seq), stay = cml_lm_sequence_length(lm, d.seq);
        if (fed > stay && cml_lm_sequence_truncate(drafter, d.draft_seq, stay)) ok = 0;
    }
    if (d.seq >= 0) cml_lm_sequence_close(lm, d.seq);
    if (d.draft_seq >= 0) cml_lm_sequence_close(drafter, d.draft_seq);
    cml_lm_keep_behind(drafter, 0);
    cmlb200_free(d.d_probabilities);
    clock_gettime(CLOCK_MONOTONIC, &t1);
    if (!ok) { cml_generation_result_free(res); return NULL; }
    res->num_tokens = n;
    const double ms = (double)(t1.tv_sec - t0.tv_sec) * 1e3 + (double)(t1.tv_nsec - t0.tv_nsec) / 1e6;
    res->total_time_ms = (float)ms;
    if (ms > 0.0) res->tokens_per_second = (float)((n - num_tokens) * 1e3 / ms);
    if (cml_lm_tokenizer(lm)) res->text = cml_tokenizer_decode(cml_lm_tokenizer(lm), res->token_ids, n);
    if (stats) *stats = s;
    return res;
}
