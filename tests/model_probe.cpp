// Test harness: the engine's model with its sizes set and nothing loaded, so
// that the range checks of its calls run on the CPU. A call that passes them
// ends at its first device call, which has no device (or only null buffers) to
// work on. Built by tests/test_host_ranges.py with g++ against the built engine.
#include <cstring>
#include <exception>
#include <string>
#include <vector>

// all that model.hpp includes, before its own members are opened
#include <map>
#include <memory>

#include "config.hpp"
#include "device.hpp"
#include "safetensors.hpp"
#include "speculative.hpp"
#include "tensor.hpp"
#define private public
#include "model.hpp"
#undef private

// call 0 forward_batch(a tokens at b), 1 steps(a after b), 2 tokens(a from b),
// 3 generate(prompt of a, b new), 4 score(a tokens at b), 5 last_logits(of a),
// 6 score(2 tokens at 0 over a vocabulary of a, b alternatives). The error's text.
extern "C" void model_ranges(int call, int max_seq, int a, int b, char* err, int n) {
    qlm::DecoderModel m;
    m.max_seq_ = max_seq;
    m.max_batch_ = m.run_B_ = 1;
    m.ld_tokens_ = max_seq + 1;
    m.cfg_.vocab_size = 8;
    const std::vector<int> some(64, 1);
    std::vector<int> out(64);
    std::string text = "no error";
    try {
        if (call == 0) m.forward_batch(some.data(), a, b, nullptr, nullptr);
        if (call == 1) m.run_steps_ = b, m.steps(a, false);
        if (call == 2) m.tokens(0, b, a, out.data());
        if (call == 3) m.generate(some.data(), 1, a, b, out.data(), nullptr);
        if (call == 4) m.score(some.data(), a, b, 0, nullptr, nullptr, nullptr, nullptr);
        if (call == 5) m.last_logits(a, reinterpret_cast<float*>(out.data()));
        if (call == 6) {
            m.cfg_.vocab_size = a;
            m.score(some.data(), 2, 0, b, nullptr, nullptr, out.data(),
                    reinterpret_cast<float*>(out.data()));
        }
    } catch (const std::exception& e) {
        text = e.what();
    }
    std::strncpy(err, text.c_str(), (size_t)n - 1);
    err[n - 1] = 0;
}
