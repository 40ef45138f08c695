// One transformer block on the host layer, trained and then served.
//
//   q = rotary(norm(x Wq)),  k = rotary(norm(x Wk)),  v = x Wv            HeadNormRotary on MatrixMultiply
//   y = norm(x + attention(q, k, v) Wo + gated(x W13) W2)                 Attention, MatrixMultiplyGated, LayerNorm
//
// Training: packed sequences of different lengths, one among them a single token, towards the outputs of another block of the
// same form.  The two branches read x side by side, so that every node but the leaves has one consumer: the executor's backward pass
// visits nodes breadth first (a node whose output is read at two depths would pass its gradient on before it is whole).
// Serving: the trained block's keys and values go into a cache with room for `CAPACITY` tokens a sequence; half of each
// sequence is read at once, the rest token by token, and the outputs must be those of the whole pass.  Then the same in 8-bit integers: products of
// quantised rows with weights laid out once, and a cache of 8-bit pages (the gated product, which has no 8-bit form, stays as it is).
//
//   deep8_transformer_block [steps]     exit code 0 if the loss fell below half and serving agrees, in 8 bits within what codes are off by
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <map>
#include <numeric>
#include <random>

#include "deep8/Deep8.h"

using namespace Deep8;

namespace {

const int WIDTH = 128, HEADS = 4, KV_HEADS = 2, DIM = 32, HIDDEN = 192, CAPACITY = 96;
const std::vector<int> LENGTHS = {37, 1, 90};

struct Block {
    Variable *wq, *wk, *wv, *wo, *w13, *w2, *qNorm, *kNorm, *outNorm, *outBias;

    Block(Executor *e, bool train) {
        auto weight = [&](size_t rows, size_t cols) {
            Variable &v = parameter(e, {rows, cols}, train);
            v.gaussian(0.f, 1.f / std::sqrt((float)rows));
            return &v;
        };
        wq = weight(WIDTH, HEADS * DIM), wk = weight(WIDTH, KV_HEADS * DIM), wv = weight(WIDTH, KV_HEADS * DIM);
        wo = weight(HEADS * DIM, WIDTH), w13 = weight(WIDTH, 2 * HIDDEN), w2 = weight(HIDDEN, WIDTH);
        qNorm = &parameter(e, {DIM}, train), kNorm = &parameter(e, {DIM}, train);
        qNorm->one(), kNorm->one();
        outNorm = &parameter(e, {WIDTH}, train), outBias = &parameter(e, {WIDTH}, train);
        outNorm->one(), outBias->zero();
    }

    Variable &operator()(Variable &x, Variable &positions, Variable &starts, Variable &table) {
        Variable &q = headNormRotary(x * *wq, *qNorm, positions, table, HEADS);
        Variable &k = headNormRotary(x * *wk, *kNorm, positions, table, KV_HEADS);
        Variable &v = x * *wv;
        Variable &seen = attention(q, k, v, starts, starts, HEADS, KV_HEADS) * *wo;
        return layerNorm(x + seen + matrixMultiplyGated(x, *w13) * *w2, *outNorm, *outBias);
    }
};

Tensor tensor(Device *dev, size_t rows, size_t cols, DType type = DType::Float32) {
    Shape shape(std::vector<size_t>{rows, cols});
    const ElementType et = ElementType::from(type);
    const size_t bytes = et.byteWidth * shape.size();
    void *ptr = dev->malloc(bytes);
    size_t *ref = (size_t *)dev->mallocCPU(sizeof(size_t));
    TensorStorage storage(ptr, ref, bytes, dev);
    return Tensor(storage, 0, shape, et);
}

// The block served: the steps that a serving of its own kind has differently are `products` and `see`.
struct Server {
    Block &block;
    Device *dev;
    Tensor table;
    std::vector<int> held;  // tokens of each sequence in the cache

    Server(Block &b, Device *d, Tensor t) : block(b), dev(d), table(t), held(LENGTHS.size(), 0) {}
    virtual ~Server() {}

    // z[i] = x w[i]
    virtual void products(const Tensor &x, const std::vector<Variable *> &w, const std::vector<Tensor *> &z) = 0;
    // counts[s] tokens of each sequence go into the cache, and o is what their queries see of it
    virtual void see(const std::vector<int> &counts, const Tensor &q, const Tensor &k, const Tensor &v, Tensor &o) = 0;

    Tensor ints(const std::vector<int> &v) {
        Tensor t = tensor(dev, 1, v.size(), DType::Int32);
        dev->copyFromCPUToGPU(v.data(), t.raw(), t.byteCount());
        return t;
    }

    // the next counts[s] tokens of each sequence, packed in x; their outputs in y
    void next(const std::vector<int> &counts, const std::vector<float> &x, std::vector<float> &y) {
        std::vector<int> positions;
        for (size_t s = 0; s < counts.size(); ++s)
            for (int i = 0; i < counts[s]; ++i) positions.push_back(held[s] + i);
        const size_t n = positions.size();
        Tensor in = tensor(dev, n, WIDTH), q = tensor(dev, n, HEADS * DIM), k = tensor(dev, n, KV_HEADS * DIM), v = tensor(dev, n, KV_HEADS * DIM);
        Tensor o = tensor(dev, n, HEADS * DIM), h = tensor(dev, n, HIDDEN), a = tensor(dev, n, WIDTH), b = tensor(dev, n, WIDTH);
        Tensor at = ints(positions);
        dev->copyFromCPUToGPU(x.data(), in.raw(), in.byteCount());
        products(in, {block.wq, block.wk, block.wv}, {&q, &k, &v});
        Math::HeadNormRotary(q, &block.qNorm->value, &at, &table, q, HEADS);
        Math::HeadNormRotary(k, &block.kNorm->value, &at, &table, k, KV_HEADS);
        see(counts, q, k, v, o);
        for (size_t s = 0; s < counts.size(); ++s) held[s] += counts[s];
        products(o, {block.wo}, {&a});
        Math::MatrixMultiplyGated(in, block.w13->value, nullptr, h);
        products(h, {block.w2}, {&b});
        Math::Add(in, a, a);
        Math::Add(a, b, a);
        Math::LayerNorm(a, &block.outNorm->value, &block.outBias->value, a);
        y.resize(n * WIDTH);
        dev->copyFromGPUToCPU(a.raw(), y.data(), a.byteCount());
    }
};

// Rows of keys and values, `CAPACITY` for each sequence.
struct PlainServer : Server {
    Tensor keys, values;
    PlainServer(Block &b, Device *d, Tensor t)
        : Server(b, d, t), keys(tensor(d, LENGTHS.size() * CAPACITY, KV_HEADS * DIM)), values(tensor(d, LENGTHS.size() * CAPACITY, KV_HEADS * DIM)) {}

    void products(const Tensor &x, const std::vector<Variable *> &w, const std::vector<Tensor *> &z) override {
        for (size_t i = 0; i < w.size(); ++i) Math::MatrixMultiply(x, w[i]->value, *z[i]);
    }

    void see(const std::vector<int> &counts, const Tensor &q, const Tensor &k, const Tensor &v, Tensor &o) override {
        const size_t row = KV_HEADS * DIM * sizeof(float);
        std::vector<int> qStarts = {0}, kStarts = {0};
        for (size_t s = 0, from = 0; s < counts.size(); from += counts[s], ++s) {
            if (counts[s]) {
                const size_t to = s * CAPACITY + held[s];
                dev->copyFromGPUToGPU((byte *)k.raw() + from * row, (byte *)keys.raw() + to * row, counts[s] * row);
                dev->copyFromGPUToGPU((byte *)v.raw() + from * row, (byte *)values.raw() + to * row, counts[s] * row);
            }
            qStarts.push_back((int)from + counts[s]);
            kStarts.push_back((int)s * CAPACITY + held[s] + counts[s]);
            if (s + 1 == counts.size()) break;
            // the cache's free places count as a sequence of keys without a query
            qStarts.push_back((int)from + counts[s]);
            kStarts.push_back((int)(s + 1) * CAPACITY);
        }
        Math::Attention(q, keys, values, ints(qStarts), ints(kStarts), o, nullptr, HEADS, KV_HEADS, 1.f / std::sqrt((float)DIM));
    }
};

// Weights as 8-bit integers, laid out once, rows quantised as they come; keys and values in 8-bit pages.
struct Int8Server : Server {
    struct Codes {
        Tensor codes, scales;
    };
    std::map<Variable *, Codes> weights;
    Math::PagedCache cache;
    Tensor pages;  // the table: sequence s has pages 2 s and 2 s + 1

    Int8Server(Block &b, Device *d, Tensor t) : Server(b, d, t) {
        for (Variable *w : {b.wq, b.wk, b.wv, b.wo, b.w2}) {
            Codes c = codes(w->value.col(), w->value.row());
            Math::QuantizeColumns(w->value, c.codes, c.scales);
            weights[w] = c;
        }
        const size_t each = (CAPACITY + Math::CACHE_PAGE - 1) / Math::CACHE_PAGE, all = LENGTHS.size() * each * KV_HEADS;
        cache = Math::PagedCache{tensor(d, all * Math::CACHE_PAGE, DIM, DType::Int8), tensor(d, all, 1), tensor(d, all * DIM, Math::CACHE_PAGE, DType::Int8), tensor(d, all, 1)};
        std::vector<int> which(LENGTHS.size() * each);
        std::iota(which.begin(), which.end(), 0);
        pages = ints(which);
    }

    Codes codes(size_t rows, size_t inner) { return Codes{tensor(dev, rows, Math::Int8Pitch(inner), DType::Int8), tensor(dev, rows, 1)}; }

    void products(const Tensor &x, const std::vector<Variable *> &w, const std::vector<Tensor *> &z) override {
        Codes c = codes(x.row(), x.col());
        Math::QuantizeRows(x, c.codes, c.scales);
        for (size_t i = 0; i < w.size(); ++i) Math::MatrixMultiplyInt8(c.codes, c.scales, weights[w[i]].codes, weights[w[i]].scales, x.col(), *z[i]);
    }

    void see(const std::vector<int> &counts, const Tensor &q, const Tensor &k, const Tensor &v, Tensor &o) override {
        std::vector<int> starts = {0}, lengths;
        for (size_t s = 0; s < counts.size(); ++s) starts.push_back(starts.back() + counts[s]), lengths.push_back(held[s] + counts[s]);
        Tensor at = ints(starts), length = ints(lengths);
        Math::CacheAppend(k, v, cache, at, length, pages, KV_HEADS);
        Math::AttentionCache(q, cache, o, nullptr, at, length, pages, HEADS, KV_HEADS, 1.f / std::sqrt((float)DIM));
    }
};

}  // namespace

int main(int argc, char **argv) {
    const int steps = argc > 1 ? std::atoi(argv[1]) : 100;
    EagerExecutor executor;
    std::vector<int> first = {0}, positions;
    for (int n : LENGTHS) {
        for (int i = 0; i < n; ++i) positions.push_back(i);
        first.push_back((int)positions.size());
    }
    const size_t tokens = positions.size();

    Variable &x = *executor.addVariable(std::vector<size_t>{tokens, WIDTH}, DType::Float32, false);
    Variable &target = *executor.addVariable(std::vector<size_t>{tokens, WIDTH}, DType::Float32, false);
    Variable &at = *executor.addVariable(std::vector<size_t>{tokens}, DType::Int32, false);
    Variable &starts = *executor.addVariable(std::vector<size_t>{first.size()}, DType::Int32, false);
    Variable &table = rotaryTable(&executor, CAPACITY, DIM);
    std::vector<float> hx(tokens * WIDTH), hy(tokens * WIDTH);
    std::mt19937 gen(7);
    std::normal_distribution<float> normal;
    for (float &f : hx) f = normal(gen);
    x.feed(hx.data()), at.feed(positions.data()), starts.feed(first.data());
    {
        Block teacher(&executor, false);
        teacher(x, at, starts, table).fetch(hy.data());
        target.feed(hy.data());
        executor.clearInterimNodes();
    }

    Block block(&executor, true);
    ConstantLearningRateIterator rate(0.003f);
    AdamTrainer trainer(&rate);
    float begin = 0, end = 0;
    for (int i = 0; i <= steps; ++i) {
        Variable &loss = (block(x, at, starts, table) - target).l2NormLoss();
        loss.fetch(&end);
        if (i == 0) begin = end;
        if (i % 20 == 0) printf("step %3d  loss %.4f\n", i, end);
        backward(loss);
        if (i < steps) trainer.train(&executor);
    }

    block(x, at, starts, table).fetch(hy.data());
    executor.clearInterimNodes();
    double largest = 0;
    for (float f : hy) largest = std::max(largest, (double)std::fabs(f));
    // served: half of each sequence at once (none of the single token), the rest token by token; how far the outputs are from the whole pass's
    auto serve = [&](Server &server) {
        double worst = 0;
        std::vector<int> counts, done(LENGTHS.size(), 0);
        for (int n : LENGTHS) counts.push_back(n / 2);
        while (std::any_of(counts.begin(), counts.end(), [](int c) { return c > 0; })) {
            std::vector<float> in, out;
            for (size_t s = 0; s < counts.size(); ++s) {
                const float *from = hx.data() + (size_t)(first[s] + done[s]) * WIDTH;
                in.insert(in.end(), from, from + (size_t)counts[s] * WIDTH);
            }
            server.next(counts, in, out);
            const float *got = out.data();
            for (size_t s = 0; s < counts.size(); ++s)
                for (int i = 0; i < counts[s]; ++i, ++done[s])
                    for (int e = 0; e < WIDTH; ++e, ++got) worst = std::max(worst, (double)std::fabs(*got - hy[(size_t)(first[s] + done[s]) * WIDTH + e]));
            for (size_t s = 0; s < counts.size(); ++s) counts[s] = done[s] < LENGTHS[s] ? 1 : 0;
        }
        return worst;
    };
    PlainServer plain(block, executor.getDevice(), table.value);
    Int8Server small(block, executor.getDevice(), table.value);
    const double worst = serve(plain), worst8 = serve(small);
    printf("loss %.4f -> %.4f; served outputs differ by at most %.2e, in 8 bits by %.2e (largest output %.2f)\n", begin, end, worst, worst8, largest);
    // (fp32 sums of a few hundred terms in another order: 1e-5 of the largest output leaves room for ten roundings in a row.  8 bits: a code is off by 1 / 254
    // of its row's largest element at most, about 1 % of an ordinary one; five such products and the cache one after the other, 5 % of the largest output)
    const bool good = std::isfinite(end) && end < 0.5f * begin && worst <= 1e-5 * largest && worst8 <= 0.05 * largest;
    printf(good ? "OK\n" : "NOT OK\n");
    return good ? 0 : 1;
}
