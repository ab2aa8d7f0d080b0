// Which parameters of a model opt::Muon takes, by which scale, what a refused step leaves behind, and what is refused. Needs a GPU.
#include <NeuZephyr/Model.cuh>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <new>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

using namespace nz;
using namespace nz::data;
using namespace nz::nodes;
using namespace nz::nodes::io;
using namespace nz::nodes::calc;

static int g_failed = 0, g_checks = 0;
static std::string g_current;
#define EXPECT_TRUE(cond)                                                              \
    do {                                                                               \
        g_checks++;                                                                    \
        if (!(cond)) {                                                                 \
            g_failed++;                                                                \
            printf("  FAILED %s: %s (line %d)\n", g_current.c_str(), #cond, __LINE__); \
        }                                                                              \
    } while (0)

static const double U = std::ldexp(1.0, -24);  // half a step of fp32, relative

static std::vector<float> normal(size_t n, unsigned seed, float std = 1.f) {
    std::mt19937 gen(seed);
    std::normal_distribution<float> d(0.f, std);
    std::vector<float> v(n);
    for (auto& x : v) x = d(gen);
    return v;
}

// five Newton-Schulz steps on r x c of x, by X' = c0 X + (c1 A + c2 A A) X with A = X X^T
static std::vector<double> orthogonal(const float* g, size_t r, size_t c) {
    std::vector<double> x(g, g + r * c);
    double norm = 0;
    for (double v : x) norm += v * v;
    norm = std::sqrt(norm) + 1e-7;
    for (double& v : x) v /= norm;
    for (int step = 0; step < 5; step++) {
        std::vector<double> a(r * r), b(r * r), y(r * c);
        for (size_t i = 0; i < r; i++)
            for (size_t j = 0; j < r; j++)
                for (size_t l = 0; l < c; l++) a[i * r + j] += x[i * c + l] * x[j * c + l];
        for (size_t i = 0; i < r; i++)
            for (size_t j = 0; j < r; j++) {
                for (size_t l = 0; l < r; l++) b[i * r + j] += 2.0315 * a[i * r + l] * a[l * r + j];
                b[i * r + j] += -4.7750 * a[i * r + j] + (i == j ? 3.4445 : 0.0);
            }
        for (size_t i = 0; i < r; i++)
            for (size_t l = 0; l < r; l++)
                for (size_t j = 0; j < c; j++) y[i * c + j] += b[i * r + l] * x[l * c + j];
        x = y;
    }
    return x;
}

// |got - (before - step * orthogonal(grad))| against the size of the update. Sums of at most 288 products go through 3 * 288 / 16 + 8
// additions that cut off up to 2^-23, three products in each of five steps, and what a matrix of low rank leaves empty has that
// noise multiplied by 3.4445 a step, 198 in all: 4.4e-3. Two roundings of w beside it.
static bool updated(const std::vector<float>& got, const std::vector<float>& before, const std::vector<float>& grad, size_t batch, size_t r,
                    size_t c, double step) {
    double err = 0, size = 0, w = 0;
    for (size_t b = 0; b < batch; b++) {
        const auto o = orthogonal(&grad[b * r * c], r, c);
        for (size_t i = 0; i < r * c; i++) {
            const double want = before[b * r * c + i] - step * o[i], d = got[b * r * c + i] - want;
            err += d * d;
            size += step * o[i] * step * o[i];
            w += want * want;
        }
    }
    return std::sqrt(err) <= 4.4e-3 * std::sqrt(size) + 8 * U * std::sqrt(w);
}
static bool descended(const std::vector<float>& got, const std::vector<float>& before, const std::vector<float>& grad, double lr) {
    for (size_t i = 0; i < got.size(); i++) {
        const double step = lr * grad[i];
        if (!(std::fabs(got[i] - (before[i] - step)) <= 2 * U * (std::fabs(before[i]) + 2 * std::fabs(step)))) return false;
    }
    return true;
}

class ConvModel : public Model {
public:
    InputNode input, target;
    Node* out = nullptr;
    ConvModel(bool fused, size_t channels, size_t out_channels, size_t kernel, bool per_sample) : input({2, channels, 6, 6}), target({2, 1, 5, 1}) {
        setFused(fused);
        computeGraph.addInput(&input);
        computeGraph.addInput(&target);
        auto x = Conv2d(&input, out_channels, kernel, kernel, 1, kernel / 2, true, per_sample);
        x = LayerNorm(ReLU(x));
        out = Softmax(Linear(x, 5));
        BCELoss(out, &target);
        const auto vx = normal(2 * channels * 36, 10);
        std::vector<float> t(10, 0.f);
        t[1] = t[8] = 1.f;
        input.dataInject(vx.begin(), vx.end());
        target.dataInject(t.begin(), t.end());
        for (size_t i = 0; i < parameters().size(); i++) {
            const auto w = normal(parameters()[i]->output->size(), 20 + (unsigned)i, 0.2f);
            parameters()[i]->dataInject(w.begin(), w.end());
        }
    }
};

// Parameters in order of their making: the convolution's weight (inputs by outputs) and bias {1, 1, Ho*Wo, Cout}, gamma, beta,
// Linear's weight (outputs by inputs) and bias.
static void conv_case(bool fused, size_t channels, size_t out_channels, size_t kernel, bool per_sample) {
    ConvModel m(fused, channels, out_channels, kernel, per_sample);
    const auto& p = m.parameters();
    EXPECT_TRUE(p.size() == 6);
    if (p.size() != 6) return;
    const double lr = 0.05f, other_lr = 0.25f;
    opt::SGD sgd((float)other_lr);
    opt::Muon muon((float)lr, 0.9f, &sgd);
    m.graph().zeroGrad();
    m.forward();
    m.backward();
    std::vector<std::vector<float>> before, grad;
    for (auto* n : p) {
        before.push_back(n->output->hostData());
        grad.push_back(n->output->hostGrad());
        double size = 0;
        for (float g : grad.back()) size += std::fabs(g);
        EXPECT_TRUE(size > 0);
    }
    m.update(&muon);
    const size_t in = channels * kernel * kernel, linear_in = 36 * out_channels;
    const double conv_step = lr * std::sqrt(std::max(1.0, (double)out_channels / in)), linear_step = lr * std::sqrt(std::max(1.0, 5.0 / linear_in));
    EXPECT_TRUE(updated(p[0]->output->hostData(), before[0], grad[0], per_sample ? 2 : 1, in, out_channels, conv_step));
    EXPECT_TRUE(updated(p[4]->output->hostData(), before[4], grad[4], 1, 5, linear_in, linear_step));
    for (size_t i : {1, 2, 3, 5}) {
        EXPECT_TRUE(descended(p[i]->output->hostData(), before[i], grad[i], other_lr));
        EXPECT_TRUE(muon.exportState(p[i]).empty());
    }
    EXPECT_TRUE(muon.exportState(p[0]).size() == 1 && muon.exportState(p[4]).size() == 1);
}
static void test_convolutions() {
    for (bool fused : {true, false}) {
        conv_case(fused, 3, 4, 3, false);  // more inputs than outputs
        conv_case(fused, 3, 8, 1, false);  // more outputs than inputs
        conv_case(fused, 2, 4, 3, true);   // a weight per sample
    }
}

// Nodes put together without a Model.
static void test_nodes_of_ones_own() {
    opt::SGD sgd(0.25f);
    opt::Muon muon(0.05f, 0.9f, &sgd);
    const auto step_once = [&](InputNode& n) {
        const auto g = normal(n.output->size(), 40), w = normal(n.output->size(), 41);
        n.output->dataInject(w.begin(), w.end());
        n.output->dataInject(g.begin(), g.end(), true);
        muon.step(&n);
        return std::make_pair(w, g);
    };
    {
        // a norm's parameters shaped like a sample
        InputNode x({2, 3, 4, 5}, true), gamma({1, 3, 4, 5}, true), beta({1, 3, 4, 5}, true);
        LayerNormNode norm(&x, &gamma, &beta);
        for (InputNode* n : {&gamma, &beta}) {
            const auto v = step_once(*n);
            EXPECT_TRUE(descended(n->output->hostData(), v.first, v.second, 0.25));
        }
    }
    {
        // a Linear bias shaped like a matrix, and its weight
        InputNode x({2, 1, 7, 1}), w({1, 1, 12, 7}, true), bias({1, 1, 3, 4}, true);
        LinearNode linear(&x, &w, &bias, false);
        const auto v = step_once(bias), u = step_once(w);
        EXPECT_TRUE(descended(bias.output->hostData(), v.first, v.second, 0.25));
        EXPECT_TRUE(updated(w.output->hostData(), u.first, u.second, 1, 12, 7, 0.05f * std::sqrt(12.0 / 7)));
    }
    {
        // a role that is given stays
        InputNode x({2, 1, 7, 1}), w({1, 1, 12, 7}, true);
        w.role = ParameterRole::NoMatrix;
        LinearNode linear(&x, &w, nullptr, false);
        const auto v = step_once(w);
        EXPECT_TRUE(descended(w.output->hostData(), v.first, v.second, 0.25));
    }
}

// The roles go with a saved graph: both go on with the same bits.
static void test_saved_graph() {
    const char* path = "/tmp/nz_muon_tests_graph.json";
    for (bool fused : {true, false}) {
        ConvModel m(fused, 3, 8, 1, false);
        opt::Adam adam(0.01f, 0.9f, 0.999f), adam2(0.01f, 0.9f, 0.999f);
        opt::Muon muon(0.05f, 0.9f, &adam), muon2(0.05f, 0.9f, &adam2);
        for (int i = 0; i < 2; i++) {
            m.graph().zeroGrad();
            m.forward();
            m.backward();
            if (i == 0) m.update(&muon);
        }
        m.graph().save(path, &muon);
        graph::ComputeGraph g;
        g.load(path, &muon2);
        m.update(&muon);
        g.update(&muon2);
        const auto &a = m.graph().getNodes(), &b = g.getNodes();
        EXPECT_TRUE(a.size() == b.size());
        size_t parameters = 0;
        for (size_t i = 0; i < a.size() && i < b.size(); i++) {
            if (!a[i]->inputs.empty() || !a[i]->output->requiresGrad()) continue;
            parameters++;
            EXPECT_TRUE(a[i]->attributes() == b[i]->attributes());
            EXPECT_TRUE(a[i]->output->hostData() == b[i]->output->hostData());
            EXPECT_TRUE(muon.exportState(a[i]) == muon2.exportState(b[i]));
        }
        EXPECT_TRUE(parameters == 6);
        EXPECT_TRUE(muon2.exportState(b[1]) == muon.exportState(a[1]));
    }
    remove(path);
}

// A graph's update that is refused leaves everything as it was; one that breaks off does not leave the other optimizer in
// the middle of a batch, where its next step would wait for an end that never comes.
static void test_refused_updates() {
    for (int kind = 0; kind < 3; kind++) {
        // 0: a slice of a matrix, 1: nobody for the vector, 2: more matrices than the operator takes (found in the step itself)
        InputNode w({1, kind == 2 ? 70000u : 1u, 2, 3}, true), bias({1, 1, 40, 1}, true), fresh({1, 1, 40, 1}, true);
        const auto v = normal(40, 50), g = normal(40, 51);
        for (InputNode* n : {&bias, &fresh}) {
            n->output->dataInject(v.begin(), v.end());
            n->output->dataInject(g.begin(), g.end(), true);
        }
        w.output->fill(0.5f);
        w.output->zeroGrad();
        opt::Adam adam(0.01f, 0.9f, 0.999f), alone(0.01f, 0.9f, 0.999f);
        opt::Muon muon(0.02f, 0.95f, kind == 1 ? nullptr : &adam);
        if (kind == 0) muon.setSlice(&w, 0, 3);
        graph::ComputeGraph graph;
        graph.addInput(&bias);
        graph.addInput(&w);
        bool threw = false, exchanged = false;
        try {
            graph.update(&muon, [&] { exchanged = true; });
        } catch (const std::exception&) {
            threw = true;
        }
        EXPECT_TRUE(threw && exchanged == (kind == 2));
        EXPECT_TRUE(bias.output->hostData() == v && w.output->hostData() == std::vector<float>(w.output->size(), 0.5f));
        EXPECT_TRUE(adam.counter() == 0);
        // the other optimizer's own steps run at once
        adam.step(&fresh);
        const auto got = fresh.output->hostData();
        fresh.output->dataInject(v.begin(), v.end());
        alone.step(&fresh);
        EXPECT_TRUE(got != v && got == fresh.output->hostData());
        // and so does the graph's update once its cause is gone
        if (kind == 0) {
            muon.setSlice(&w, 0, 0);
            graph.update(&muon);
            EXPECT_TRUE(bias.output->hostData() != v);
        }
    }
}

// One node cannot be both of a norm's parameters: two sums would be added to one gradient at a time.
static void test_norm_of_one_parameter() {
    InputNode x({2, 1, 8, 1}, true), g({1, 1, 8, 1}, true);
    bool threw = false;
    try {
        LayerNormNode norm(&x, &g, &g);
    } catch (const std::invalid_argument&) {
        threw = true;
    }
    EXPECT_TRUE(threw);
}

// A parameter at the address of one that is gone, of another size: it has a state of its own.
static void test_address_taken_again() {
    alignas(InputNode) unsigned char place[sizeof(InputNode)];
    opt::Adam adam(0.01f, 0.9f, 0.999f);
    opt::Muon muon(0.05f, 0.9f, &adam);
    const size_t sides[][2] = {{4, 6}, {40, 70}, {70, 40}, {300, 1}, {4, 1}};
    for (const auto& hw : sides) {
        const size_t h = hw[0], w = hw[1];
        auto* n = new (place) InputNode({1, 1, h, w}, true);
        const auto v = normal(h * w, 60), g = normal(h * w, 61);
        n->output->dataInject(v.begin(), v.end());
        n->output->dataInject(g.begin(), g.end(), true);
        muon.step(n);
        const auto got = n->output->hostData(), state = muon.exportState(n)[0];
        EXPECT_TRUE(state.size() == h * w);
        if (w > 1) {
            EXPECT_TRUE(updated(got, v, g, 1, h, w, 0.05f * std::sqrt(std::max(1.0, (double)h / w))));
            EXPECT_TRUE(state == g);  // the first step's momentum
        } else {
            // Adam's first moment after one step: (1 - 0.9) g
            double worst = 0;
            for (size_t i = 0; i < h; i++) worst = std::max(worst, std::fabs(state[i] - (1.0 - 0.9f) * g[i]));
            EXPECT_TRUE(worst <= 4 * U * 4);
        }
        n->~InputNode();
    }
}

int main() {
    const struct { const char* name; void (*fn)(); } tests[] = {
        {"convolutions", test_convolutions}, {"nodes_of_ones_own", test_nodes_of_ones_own}, {"saved_graph", test_saved_graph},
        {"refused_updates", test_refused_updates}, {"norm_of_one_parameter", test_norm_of_one_parameter},
        {"address_taken_again", test_address_taken_again},
    };
    for (auto& t : tests) {
        g_current = t.name;
        const int before = g_failed;
        try {
            t.fn();
        } catch (const std::exception& e) {
            g_failed++;
            printf("  EXCEPTION in %s: %s\n", t.name, e.what());
        }
        printf("[%s] %s\n", g_failed == before ? "  OK  " : "FAILED", t.name);
    }
    cuStrm::StreamManager<float>::Instance().sync();
    int status = 0;
    nzb_device_status(&status);
    printf("%d checks, %d failures, device status %d\n", g_checks, g_failed, status);
    return (g_failed || status) ? 1 : 0;
}
