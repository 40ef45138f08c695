// One transformer block on the host layer, trained and then served.
//
//   q = rotary(norm(x Wq)),  k = rotary(norm(x Wk)),  v = x Wv            HeadNormRotary on MatrixMultiply
//   y = x + attention(q, k, v) Wo + gated(x W13) W2                       Attention, MatrixMultiplyGated
//
// Training: packed sequences of different lengths, one among them a single token, towards the outputs of another block of the
// same form.  The two branches read x side by side, so that every node but the leaves has one consumer: the executor's backward pass
// visits nodes breadth first (a node whose output is read at two depths would pass its gradient on before it is whole).
// Serving: the trained block's keys and values go into a cache with room for `CAPACITY` tokens a sequence; half of each
// sequence is read at once, the rest token by token, and the outputs must be those of the whole pass.
//
//   deep8_transformer_block [steps]     exit code 0 if the loss fell below half and serving agrees
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <random>

#include "deep8/Deep8.h"

using namespace Deep8;

namespace {

const int WIDTH = 128, HEADS = 4, KV_HEADS = 2, DIM = 32, HIDDEN = 192, CAPACITY = 96;
const std::vector<int> LENGTHS = {37, 1, 90};

struct Block {
    Variable *wq, *wk, *wv, *wo, *w13, *w2, *qNorm, *kNorm;

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
    }

    Variable &operator()(Variable &x, Variable &positions, Variable &starts, Variable &table) {
        Variable &q = headNormRotary(x * *wq, *qNorm, positions, table, HEADS);
        Variable &k = headNormRotary(x * *wk, *kNorm, positions, table, KV_HEADS);
        Variable &v = x * *wv;
        Variable &seen = attention(q, k, v, starts, starts, HEADS, KV_HEADS) * *wo;
        return x + seen + matrixMultiplyGated(x, *w13) * *w2;
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

// The block with a cache of keys and values per sequence.
struct Server {
    Block &block;
    Device *dev;
    Tensor table, keys, values;
    std::vector<int> held;  // tokens of each sequence in the cache

    Server(Block &b, Device *d, Tensor t)
        : block(b), dev(d), table(t), keys(tensor(d, LENGTHS.size() * CAPACITY, KV_HEADS * DIM)),
          values(tensor(d, LENGTHS.size() * CAPACITY, KV_HEADS * DIM)), held(LENGTHS.size(), 0) {}

    Tensor ints(const std::vector<int> &v) {
        Tensor t = tensor(dev, 1, v.size(), DType::Int32);
        dev->copyFromCPUToGPU(v.data(), t.raw(), t.byteCount());
        return t;
    }

    // the next counts[s] tokens of each sequence, packed in x; their outputs in y
    void next(const std::vector<int> &counts, const std::vector<float> &x, std::vector<float> &y) {
        std::vector<int> positions, qStarts = {0}, kStarts = {0};
        for (size_t s = 0; s < counts.size(); ++s) {
            for (int i = 0; i < counts[s]; ++i) positions.push_back(held[s] + i);
            qStarts.push_back((int)positions.size());
            kStarts.push_back((int)s * CAPACITY + held[s] + counts[s]);
            if (s + 1 == counts.size()) break;
            // the cache's free places count as a sequence of keys without a query
            qStarts.push_back((int)positions.size());
            kStarts.push_back((int)(s + 1) * CAPACITY);
        }
        const size_t n = positions.size();
        Tensor in = tensor(dev, n, WIDTH), q = tensor(dev, n, HEADS * DIM), k = tensor(dev, n, KV_HEADS * DIM), v = tensor(dev, n, KV_HEADS * DIM);
        Tensor o = tensor(dev, n, HEADS * DIM), h = tensor(dev, n, HIDDEN), a = tensor(dev, n, WIDTH), b = tensor(dev, n, WIDTH);
        Tensor at = ints(positions), qs = ints(qStarts), ks = ints(kStarts);
        dev->copyFromCPUToGPU(x.data(), in.raw(), in.byteCount());
        Math::MatrixMultiply(in, block.wq->value, q);
        Math::MatrixMultiply(in, block.wk->value, k);
        Math::MatrixMultiply(in, block.wv->value, v);
        Math::HeadNormRotary(q, &block.qNorm->value, &at, &table, q, HEADS);
        Math::HeadNormRotary(k, &block.kNorm->value, &at, &table, k, KV_HEADS);
        const size_t row = KV_HEADS * DIM * sizeof(float);
        for (size_t s = 0, from = 0; s < counts.size(); from += counts[s], ++s) {
            if (!counts[s]) continue;
            const size_t to = s * CAPACITY + held[s];
            dev->copyFromGPUToGPU((byte *)k.raw() + from * row, (byte *)keys.raw() + to * row, counts[s] * row);
            dev->copyFromGPUToGPU((byte *)v.raw() + from * row, (byte *)values.raw() + to * row, counts[s] * row);
            held[s] += counts[s];
        }
        Math::Attention(q, keys, values, qs, ks, o, nullptr, HEADS, KV_HEADS, 1.f / std::sqrt((float)DIM));
        Math::MatrixMultiply(o, block.wo->value, a);
        Math::MatrixMultiplyGated(in, block.w13->value, nullptr, h);
        Math::MatrixMultiply(h, block.w2->value, b);
        Math::Add(in, a, a);
        Math::Add(a, b, a);
        y.resize(n * WIDTH);
        dev->copyFromGPUToCPU(a.raw(), y.data(), a.byteCount());
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
    Server server(block, executor.getDevice(), table.value);
    double worst = 0, largest = 0;
    std::vector<int> counts, done(LENGTHS.size(), 0);
    for (int n : LENGTHS) counts.push_back(n / 2);  // half of each sequence at once (none of the single token)
    for (int calls = 0; std::any_of(counts.begin(), counts.end(), [](int c) { return c > 0; }); ++calls) {
        std::vector<float> in, out;
        for (size_t s = 0; s < counts.size(); ++s) {
            const float *from = hx.data() + (size_t)(first[s] + done[s]) * WIDTH;
            in.insert(in.end(), from, from + (size_t)counts[s] * WIDTH);
        }
        server.next(counts, in, out);
        const float *got = out.data();
        for (size_t s = 0; s < counts.size(); ++s)
            for (int i = 0; i < counts[s]; ++i, ++done[s])
                for (int e = 0; e < WIDTH; ++e, ++got) {
                    const float want = hy[(size_t)(first[s] + done[s]) * WIDTH + e];
                    worst = std::max(worst, (double)std::fabs(*got - want));
                    largest = std::max(largest, (double)std::fabs(want));
                }
        for (size_t s = 0; s < counts.size(); ++s) counts[s] = done[s] < LENGTHS[s] ? 1 : 0;
    }
    printf("loss %.4f -> %.4f; served outputs differ by at most %.2e (largest output %.2f)\n", begin, end, worst, largest);
    // (fp32 sums of a few hundred terms in another order: 1e-5 of the largest output leaves room for ten roundings in a row)
    const bool good = std::isfinite(end) && end < 0.5f * begin && worst <= 1e-5 * largest;
    printf(good ? "OK\n" : "NOT OK\n");
    return good ? 0 : 1;
}
