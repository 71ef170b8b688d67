/* main.c -- engine CLI with the reference's flags (engine/src/main.c:28-109):
 *   shukuchi <model.gguf> [--prompt "..."] [--max-tokens N] [--tokens 1,2,3]
 * SHUKUCHI_PREFETCH_DEPTH sets the loader depth (default 3; 0 -> 2).  Tokens
 * are printed as "<id>text"; the streaming statistics line follows on stderr.
 * --tokens (an addition) feeds token ids instead of prompt text; --temperature,
 * --top-k, --top-p, --min-p and --seed (additions) draw the tokens at random. */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/resource.h>

#include "engine.h"

int main(int argc, char **argv) {
    if (argc < 2) {
        fprintf(stderr,
                "Usage: %s <model.gguf> [--prompt \"...\"] [--max-tokens N] [--tokens 1,2,3]\n"
                "       [--temperature T] [--top-k K] [--top-p P] [--min-p P] [--seed S]\n",
                argv[0]);
        return 1;
    }
    uint32_t max_tokens = 16;
    const char *prompt = NULL, *tokens = NULL;
    float temperature = 0.f, top_p = 1.f, min_p = 0.f;
    int top_k = 0;
    uint64_t seed = 0;
    for (int i = 2; i + 1 < argc; ++i) {
        if (strcmp(argv[i], "--max-tokens") == 0) max_tokens = (uint32_t)strtoul(argv[++i], NULL, 10);
        else if (strcmp(argv[i], "--prompt") == 0) prompt = argv[++i];
        else if (strcmp(argv[i], "--tokens") == 0) tokens = argv[++i];
        else if (strcmp(argv[i], "--temperature") == 0) temperature = strtof(argv[++i], NULL);
        else if (strcmp(argv[i], "--top-k") == 0) top_k = (int)strtol(argv[++i], NULL, 10);
        else if (strcmp(argv[i], "--top-p") == 0) top_p = strtof(argv[++i], NULL);
        else if (strcmp(argv[i], "--min-p") == 0) min_p = strtof(argv[++i], NULL);
        else if (strcmp(argv[i], "--seed") == 0) seed = strtoull(argv[++i], NULL, 10);
    }
    uint32_t depth = 3;
    const char *env = getenv("SHUKUCHI_PREFETCH_DEPTH");
    if (env && *env) {
        depth = (uint32_t)strtoul(env, NULL, 10);
        if (depth == 0) depth = 2;
    }
    struct engine_config cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.n_threads = 4;
    cfg.batch_size = 1;
    cfg.prefetch_depth = depth;
    cfg.kv_block_size = 32;
    engine_handle_t *h = engine_open(argv[1], &cfg);
    if (!h) {
        fprintf(stderr, "engine: failed to open model\n");
        return 1;
    }
    if (engine_set_sampling(h, temperature, top_k, top_p, min_p, seed) != 0) {
        fprintf(stderr, "engine: bad sampling settings\n");
        engine_close(h);
        return 1;
    }
    int rc;
    if (tokens) {
        uint32_t ids[4096];
        uint32_t n = 0;
        for (const char *p = tokens; *p && n < 4096;) {
            char *end;
            ids[n++] = (uint32_t)strtoul(p, &end, 10);
            p = (*end == ',') ? end + 1 : end;
            if (end == p && *p) break;
        }
        rc = engine_generate_ids(h, ids, n, max_tokens, NULL, NULL) < 0;
        if (!rc) printf("%s\n", engine_get_output(h));
    } else {
        if (prompt) engine_set_prompt(h, prompt);
        rc = engine_generate(h, max_tokens) != 0;
    }
    struct streaming_stats st;
    if (engine_get_streaming_stats(h, &st) == 0)
        fprintf(stderr,
                "streaming_stats: layer_loads=%llu layer_bytes_read=%llu max_layer_size=%zu peak_buffer_usage=%zu "
                "peak_rss=%zu max_concurrent_buffers=%u prefetch_hits=%u prefetch_misses=%u\n",
                (unsigned long long)st.layer_loads, (unsigned long long)st.layer_bytes_read, st.max_layer_size,
                st.peak_buffer_usage, st.peak_rss, st.max_concurrent_buffers, st.prefetch_hits,
                st.prefetch_misses);
    engine_report(h); /* engine/src/main.c:106 metal_ops_report() */
    engine_close(h);
    struct rusage ru;
    if (getrusage(RUSAGE_SELF, &ru) == 0) fprintf(stderr, "peak_rss_mb=%.2f\n", (double)ru.ru_maxrss / 1024.0);
    if (rc) fprintf(stderr, "engine: generation failed\n");
    return rc;
}
