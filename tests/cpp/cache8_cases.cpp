// The C++ host mirror's 8-bit caches, windows and rotary positions with several axes (include/fusor_cuda.hpp).
// Usage: cache8_cases            -> runs on GPU 0, exit code 0 on success
//        cache8_cases --no-gpu   -> host-only checks
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "fusor_cuda.hpp"

using namespace fusor_cuda;
static int failures = 0;
#define CHECK(cond)                                                        \
    do {                                                                   \
        if (!(cond)) {                                                     \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);  \
            ++failures;                                                    \
        }                                                                  \
    } while (0)
template <class F>
static bool throws(F f) {
    try {
        f();
    } catch (const std::exception&) {
        return true;
    }
    return false;
}

// Values that an 8-bit row holds exactly: whole numbers below 64 with a 64 among them (step 1)
static std::vector<float> rows(int64_t heads, int64_t n, int64_t d, int seed) {
    std::vector<float> x(heads * n * d);
    for (int64_t r = 0; r < heads * n; ++r)
        for (int64_t i = 0; i < d; ++i) x[r * d + i] = i == (r + seed) % d ? 64.0f : (float)((r * 7 + i * 3 + seed) % 41 - 20);
    return x;
}

static void host_only() {
    CHECK(throws([] { KvCache(2, 8, FUSOR_CUDA_F16); }));
    CHECK(!throws([] { KvCache(2, 8, FUSOR_CUDA_I8); }));
    LlamaCacheConfig config;
    config.n_layer = 2;
    config.context_length = 16;
    config.cache_dtype = FUSOR_CUDA_I8;
    CHECK(LlamaCache(config).blocks.size() == 2);
    RopeAxes axes;
    axes.axis_of_pair = {0, 1, 1};
    CHECK(throws([&] { axes.view({1, 1, 1, 8}); }));  // four pairs
    axes.axis_of_pair = {0, 1, 1, 0};
    axes.n_axes = 2;
    CHECK(axes.view({3, 2, 5, 8}).axis_stride == 5 && axes.view({3, 2, 5, 8}).batch_stride == 0);
    axes.per_sequence = true;
    CHECK(axes.view({3, 2, 5, 8}).axis_stride == 15 && axes.view({3, 2, 5, 8}).batch_stride == 5);
}

static void caches(const DevicePtr& dev, int32_t dtype) {
    const int64_t H = 2, D = 64;
    KvCache cache(2, 20, dtype);
    const auto a = rows(2 * H, 20, D, 0), b = rows(2 * H, 20, D, 5);
    const auto T = [&](const std::vector<float>& x, int64_t batch, int64_t n, int64_t h = 2) { return Tensor<4>::from_slice(dev, {batch, h, n, D}, x); };
    cache.append(dev, T(a, 2, 20), T(b, 2, 20));
    CHECK(cache.dense(DType::F32).first.as_slice() == a && cache.dense(DType::F32).second.as_slice() == b);
    // refused on a full window: another batch; a head_dim without kernels: as it was
    const auto one = rows(H, 1, D, 9);
    CHECK(throws([&] { cache.append(dev, T(one, 1, 1), T(one, 1, 1)); }));
    CHECK(throws([&] { cache.append(dev, Tensor<4>::from_slice(dev, {2, 2, 1, 32}, rows(4, 1, 32, 0)), Tensor<4>::from_slice(dev, {2, 2, 1, 32}, rows(4, 1, 32, 0))); }));
    CHECK(cache.current_seq_len() == 20);
    CHECK(cache.dense(DType::F32).first.as_slice() == a && cache.dense(DType::F32).second.as_slice() == b);
    // one more row, then a prompt longer than the window, then other heads
    const auto next = rows(2 * H, 1, D, 3), prompt = rows(2 * H, 27, D, 4);
    cache.append(dev, T(next, 2, 1), T(next, 2, 1));
    const auto got = cache.dense(DType::F32).first.as_slice();
    bool same = cache.current_seq_len() == 20;
    for (int64_t h = 0; h < 2 * H; ++h)
        for (int64_t i = 0; i < 20 * D; ++i) same = same && got[h * 20 * D + i] == (i < 19 * D ? a[(h * 20 + 1) * D + i] : next[h * D + i - 19 * D]);
    CHECK(same);
    cache.append(dev, T(prompt, 2, 27), T(prompt, 2, 27));
    const auto last = cache.dense(DType::F32).second.as_slice();
    same = cache.current_seq_len() == 20;
    for (int64_t h = 0; h < 2 * H; ++h)
        for (int64_t i = 0; i < 20 * D; ++i) same = same && last[h * 20 * D + i] == prompt[(h * 27 + 7) * D + i];
    CHECK(same);
    const auto other = rows(1, 5, D, 2);
    cache.append(dev, T(other, 1, 5, 1), T(other, 1, 5, 1));
    CHECK(cache.current_seq_len() == 5 && cache.dense(DType::F32).first.as_slice() == other);
    // a key far above the others: its value
    std::vector<float> q(D, 0.0f);
    for (int64_t i = 0; i < D; ++i) q[i] = other[2 * D + i] * 0.25f;
    const auto o = cache.attend(Tensor<4>::from_slice(dev, {1, 1, 1, D}, q), 1.0f, std::nullopt).as_slice();
    for (int64_t i = 0; i < D; ++i) CHECK(std::fabs(o[i] - other[2 * D + i]) <= 1e-4f);
    cache.reset();
    CHECK(cache.current_seq_len() == 0);
}

static void positions(const DevicePtr& dev) {
    const int64_t D = 8, n = 3, B = 2, C = 10;
    std::vector<float> cos(C * D / 2), sin(C * D / 2), x(B * 2 * n * D), y(B * n * D);
    for (size_t i = 0; i < cos.size(); ++i) cos[i] = (float)((int)(i % 5) - 2), sin[i] = (float)((int)(i % 7) - 3);
    for (size_t i = 0; i < x.size(); ++i) x[i] = (float)((int)(i * 11 % 23) - 11);
    for (size_t i = 0; i < y.size(); ++i) y[i] = (float)((int)(i * 5 % 19) - 9);
    const uint32_t ids[2 * B * n] = {0, 1, 2, 3, 4, 5, 9, 8, 7, 6, 5, 4};  // [axis][B][n]
    auto on_device = Tensor<2>::from_slice(dev, {2, B * n}, std::vector<float>(2 * B * n));  // (12 words of 4 bytes)
    dev->check(fusor_cuda_buffer_upload(dev->raw(), on_device.data(), ids, sizeof ids));
    dev->synchronize();
    RopeAxes axes;
    axes.ids = static_cast<const uint32_t*>(on_device.data());
    axes.per_sequence = true;
    axes.n_axes = 2;
    axes.axis_of_pair = {0, 1, 1, 0};
    RopeCache rope(Tensor<2>::from_slice(dev, {C, D / 2}, cos), Tensor<2>::from_slice(dev, {C, D / 2}, sin));
    const auto q = Tensor<4>::from_slice(dev, {B, 2, n, D}, x);
    const auto k = Tensor<4>::from_slice(dev, {B, 1, n, D}, y);
    for (const bool interleaved : {false, true}) {
        const auto want = [&](const std::vector<float>& in, int64_t heads) {
            std::vector<float> out(in.size());
            for (int64_t b = 0; b < B; ++b)
                for (int64_t h = 0; h < heads; ++h)
                    for (int64_t t = 0; t < n; ++t)
                        for (int64_t i = 0; i < D / 2; ++i) {
                            const int64_t at = ((b * heads + h) * n + t) * D, row = ids[(axes.axis_of_pair[i] * B + b) * n + t] * (D / 2) + i;
                            const int64_t da = at + (interleaved ? 2 * i : i), db = at + (interleaved ? 2 * i + 1 : i + D / 2);
                            out[da] = in[da] * cos[row] - in[db] * sin[row];
                            out[db] = in[da] * sin[row] + in[db] * cos[row];
                        }
            return out;
        };
        const auto both = rope.forward_axes(q, k, axes, interleaved);
        CHECK(both.first.as_slice() == want(x, 2) && both.second.as_slice() == want(y, 1));
        CHECK(rope_axes(q, rope.cos(), rope.sin(), axes, interleaved).as_slice() == want(x, 2));
    }
    axes.axis_of_pair[3] = 2;
    CHECK(throws([&] { rope.forward_axes(q, k, axes); }));
    CHECK(throws([&] { rope.forward_axes(q, Tensor<4>::from_slice(dev, {B, 1, 1, D}, std::vector<float>(B * D)), axes); }));
}

int main(int argc, char** argv) {
    host_only();
    if (!(argc > 1 && std::strcmp(argv[1], "--no-gpu") == 0)) {
        try {
            const DevicePtr dev = Device::gpu(0);
            caches(dev, FUSOR_CUDA_I8);
            caches(dev, FUSOR_CUDA_BF16);
            positions(dev);
        } catch (const std::exception& e) {
            std::printf("FAILED with exception: %s\n", e.what());
            ++failures;
        }
    }
    std::printf(failures ? "%d check(s) failed\n" : "all cache cases passed\n", failures);
    return failures ? 1 : 0;
}
