// sample.hip's launches on the CPU (hip/hip_runtime.h beside this file). SAMPLE names a copy of
// sample.hip without its inline assembly.
#include <hip/hip_runtime.h>

#include SAMPLE

#include <vector>

namespace migemm {
bool plan_only() { return false; }
int launch_status(const char *) { return 0; }
void *workspace(hipStream_t, size_t bytes, int *status, int) {
    static std::vector<char> held;
    held.assign(bytes, (char)0xa5);
    *status = 0;
    return held.data();
}
}  // namespace migemm

extern "C" int run(const void *logits, int type, int64_t ld, int rows, int vocab,
                   const float *uniforms, float temperature, int top_k, float top_p, float min_p,
                   int *tokens, float *probabilities, int order) {
    migemm::SampleArgs p{};
    p.logits = logits;
    p.type = type;
    p.ld = ld;
    p.rows = rows;
    p.vocab = vocab;
    p.uniforms = uniforms;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.tokens = tokens;
    p.probabilities = probabilities;
    cpu::order = order;
    return migemm::launch_sample(nullptr, p);
}
