// Tests of the layer norm node and the Muon optimizer of the C++ host layer against the formulas in double. Needs a GPU.
#include <NeuZephyr/Model.cuh>
#include <NeuZephyr/TensorOperations.cuh>

#include <algorithm>
#include <cmath>
#include <cstdio>
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
#define EXPECT_THROW(statement, type)   \
    do {                                \
        bool threw = false;             \
        try {                           \
            statement;                  \
        } catch (const type&) {         \
            threw = true;               \
        }                               \
        EXPECT_TRUE(threw);             \
    } while (0)

static const double U = std::ldexp(1.0, -24);  // half a step of fp32, relative

static std::vector<float> normal(size_t n, unsigned seed, float mean = 0.f, float std = 1.f) {
    std::mt19937 gen(seed);
    std::normal_distribution<float> d(mean, std);
    std::vector<float> v(n);
    for (auto& x : v) x = d(gen);
    return v;
}
static double worst(const std::vector<float>& got, const std::vector<double>& want) {
    if (got.size() != want.size()) return INFINITY;
    double w = 0;
    for (size_t i = 0; i < got.size(); i++) {
        const double d = std::fabs(got[i] - want[i]);
        if (!(d <= w)) w = d;  // a NaN stays
    }
    return w;
}

struct NormOracle {
    std::vector<double> y, dx, dgamma, dbeta;
    NormOracle(size_t n, size_t dim, const std::vector<float>& x, const std::vector<float>& g, const std::vector<float>& b,
               const std::vector<float>& dy, double eps)
        : y(n * dim), dx(n * dim), dgamma(dim), dbeta(dim) {
        for (size_t r = 0; r < n; r++) {
            const float* xr = &x[r * dim];
            double mean = 0, var = 0, s1 = 0, s2 = 0;
            for (size_t c = 0; c < dim; c++) mean += xr[c] / (double)dim;
            for (size_t c = 0; c < dim; c++) var += (xr[c] - mean) * (xr[c] - mean) / (double)dim;
            const double rstd = 1 / std::sqrt(var + eps);
            for (size_t c = 0; c < dim; c++) {
                const double h = (xr[c] - mean) * rstd, d = dy[r * dim + c];
                y[r * dim + c] = h * g[c] + b[c];
                dgamma[c] += d * h;
                dbeta[c] += d;
                s1 += d * g[c] / dim;
                s2 += d * g[c] * h / dim;
            }
            for (size_t c = 0; c < dim; c++) {
                const double h = (xr[c] - mean) * rstd;
                dx[r * dim + c] = rstd * (dy[r * dim + c] * g[c] - s1 - h * s2);
            }
        }
    }
};

static void layer_norm_case(size_t n, size_t c, size_t h, size_t w, bool overwrite) {
    const size_t dim = c * h * w;
    InputNode x({n, c, h, w}, true), gamma({1, 1, 1, dim}, true), beta({1, c, h, w}, true);
    const auto vx = normal(n * dim, 1, 0.5f, 2.f), vg = normal(dim, 2, 1.f, 0.2f), vb = normal(dim, 3), vd = normal(n * dim, 4);
    x.output->dataInject(vx.begin(), vx.end());
    gamma.output->dataInject(vg.begin(), vg.end());
    beta.output->dataInject(vb.begin(), vb.end());
    LayerNormNode norm(&x, &gamma, &beta, 1e-5f);
    norm.forward();
    NormOracle o(n, dim, vx, vg, vb, vd, 1e-5f);
    // numbers below 10 in size; sums over dim elements are joined from shares of at most 32, and a handful of roundings
    const double row_tol = 10 * 64 * U, col_tol = 10 * (n + 16) * U * std::sqrt((double)n);
    EXPECT_TRUE(worst(norm.output->hostData(), o.y) <= row_tol);
    norm.output->dataInject(vd.begin(), vd.end(), true);
    const auto before = normal(n * dim, 5);
    x.output->dataInject(before.begin(), before.end(), true);
    x.output->setGradOverwritten(overwrite);
    gamma.output->zeroGrad();
    beta.output->zeroGrad();
    norm.backward();
    auto dx = o.dx;
    if (!overwrite)
        for (size_t i = 0; i < dx.size(); i++) dx[i] += before[i];
    EXPECT_TRUE(worst(x.output->hostGrad(), dx) <= row_tol);
    EXPECT_TRUE(worst(gamma.output->hostGrad(), o.dgamma) <= col_tol);
    EXPECT_TRUE(worst(beta.output->hostGrad(), o.dbeta) <= col_tol);
    // a second pass adds to the parameters' gradients
    norm.backward();
    for (double& v : o.dgamma) v *= 2;
    EXPECT_TRUE(worst(gamma.output->hostGrad(), o.dgamma) <= 2 * col_tol);
}

// the oracle's gradients against differences of sum(dy * y), in double
static void test_oracle() {
    const size_t n = 3, dim = 7;
    auto x = normal(n * dim, 6), g = normal(dim, 7), b = normal(dim, 8);
    const auto d = normal(n * dim, 9);
    const NormOracle o(n, dim, x, g, b, d, 1e-5);
    const auto slope = [&](float& v) {
        const float mid = v, step = std::ldexp(1.f, -9);  // mid +- step are rounded: the step taken is what counts
        double sum[2], at[2];
        for (int side = 0; side < 2; side++) {
            v = mid + (side ? step : -step);
            at[side] = v;
            const NormOracle p(n, dim, x, g, b, d, 1e-5);
            sum[side] = 0;
            for (size_t i = 0; i < n * dim; i++) sum[side] += d[i] * p.y[i];
        }
        v = mid;
        return (sum[1] - sum[0]) / (at[1] - at[0]);
    };
    // the third derivative, of size 100 at the most here, times step^2 / 6
    for (size_t i = 0; i < n * dim; i++) EXPECT_TRUE(std::fabs(slope(x[i]) - o.dx[i]) <= 1e-4);
    for (size_t i = 0; i < dim; i++) EXPECT_TRUE(std::fabs(slope(g[i]) - o.dgamma[i]) <= 1e-4);
    for (size_t i = 0; i < dim; i++) EXPECT_TRUE(std::fabs(slope(b[i]) - o.dbeta[i]) <= 1e-4);
}

static void test_layer_norm() {
    layer_norm_case(5, 1, 33, 1, false);
    layer_norm_case(5, 3, 7, 11, true);
    layer_norm_case(1, 1, 64, 1, false);
    layer_norm_case(300, 4, 8, 8, true);
    // one element to a sample: its own mean, so beta comes out and no gradient goes in
    InputNode x({3, 1, 1, 1}, true), gamma({1, 1, 1, 1}, true), beta({1, 1, 1, 1}, true);
    x.output->dataInject({5.f, -2.f, 0.f});
    gamma.output->fill(2.f);
    beta.output->fill(0.25f);
    LayerNormNode norm(&x, &gamma, &beta);
    norm.forward();
    EXPECT_TRUE(norm.output->hostData() == std::vector<float>(3, 0.25f));
    norm.output->dataInject({1.f, 1.f, 1.f}, true);
    x.output->zeroGrad();
    norm.backward();
    EXPECT_TRUE(x.output->hostGrad() == std::vector<float>(3, 0.f));
}

static void test_layer_norm_refusals() {
    InputNode x({3, 2, 4, 1}, true), g({1, 1, 1, 8}, true), shorter({1, 1, 1, 7}, true);
    EXPECT_THROW(LayerNormNode(&x, &g, &shorter), std::invalid_argument);
    EXPECT_THROW(LayerNormNode(&x, &shorter, &g), std::invalid_argument);
    EXPECT_THROW(LayerNormNode(&x, &g, nullptr), std::invalid_argument);
    EXPECT_THROW(LayerNormNode(&x, &g, &g, -1.f), std::invalid_argument);
    EXPECT_THROW(LayerNormNode(&x, &g, &g, NAN), std::invalid_argument);
}

class NormModel : public Model {
public:
    InputNode input, target;
    Node* out = nullptr;
    explicit NormModel(size_t batch, bool fused = true) : input({batch, 1, 70, 1}), target({batch, 1, 8, 1}) {
        setFused(fused);
        computeGraph.addInput(&input);
        computeGraph.addInput(&target);
        auto x = Linear(&input, 96);
        x = LayerNorm(x, 1e-4f);
        x = ReLU(x);
        x = Linear(x, 80);
        x = LayerNorm(x);
        x = Linear(x, 8);
        out = Softmax(x);
        BCELoss(out, &target);
        const auto vx = normal(batch * 70, 10);
        std::vector<float> t(batch * 8, 0.f);
        for (size_t i = 0; i < batch; i++) t[i * 8 + i % 8] = 1.f;
        input.dataInject(vx.begin(), vx.end());
        target.dataInject(t.begin(), t.end());
        for (size_t i = 0; i < parameters().size(); i++) {
            auto w = normal(parameters()[i]->output->size(), 20 + (unsigned)i, 0.f, 0.1f);
            parameters()[i]->dataInject(w.begin(), w.end());
        }
    }
};

static void run_step(Model& m, opt::Optimizer* o) {
    m.graph().zeroGrad();
    m.forward();
    m.backward();
    m.update(o);
}

static void test_model_of_norms() {
    NormModel a(16), b(16, false);
    EXPECT_TRUE(a.parameters().size() == 10 && b.parameters().size() == 10);
    // the parameters of a new layer norm
    class Fresh : public Model {
    public:
        InputNode input;
        Fresh() : input({2, 3, 4, 5}) { computeGraph.addInput(&input); LayerNorm(&input); }
    } fresh;
    EXPECT_TRUE(fresh.parameters()[0]->output->hostData() == std::vector<float>(60, 1.f));
    EXPECT_TRUE(fresh.parameters()[1]->output->hostData() == std::vector<float>(60, 0.f));
    a.graph().zeroGrad();
    b.graph().zeroGrad();
    for (Model* m : {(Model*)&a, (Model*)&b}) {
        m->forward();
        m->backward();
    }
    const auto ya = a.out->output->hostData(), yb = b.out->output->hostData();
    double d = 0;
    for (size_t i = 0; i < ya.size(); i++) d = std::max(d, (double)std::fabs(ya[i] - yb[i]));
    // products of tf32 at the least: 2^-10 of numbers of size 1 after a norm, times gamma and weights of size 0.1
    EXPECT_TRUE(d <= 4e-3);
}

// rows x cols of u, five Newton-Schulz steps
static std::vector<double> orthogonal(std::vector<double> x, size_t r, size_t c) {
    double norm = 0;
    for (double v : x) norm += v * v;
    norm = std::sqrt(norm) + 1e-7;
    for (double& v : x) v /= norm;
    const bool tall = r > c;
    const auto gram = [&](const std::vector<double>& m) {
        const size_t n = tall ? c : r, k = tall ? r : c;
        std::vector<double> a(n * n);
        for (size_t i = 0; i < n; i++)
            for (size_t j = 0; j < n; j++) {
                double s = 0;
                for (size_t l = 0; l < k; l++) s += tall ? m[l * c + i] * m[l * c + j] : m[i * c + l] * m[j * c + l];
                a[i * n + j] = s;
            }
        return a;
    };
    const size_t n = tall ? c : r;
    for (int step = 0; step < 5; step++) {
        const auto a = gram(x);
        std::vector<double> p(n * n);
        for (size_t i = 0; i < n; i++)
            for (size_t j = 0; j < n; j++) {
                double s = 0;
                for (size_t l = 0; l < n; l++) s += a[i * n + l] * a[l * n + j];
                p[i * n + j] = -4.7750 * a[i * n + j] + 2.0315 * s;
            }
        for (size_t i = 0; i < n; i++) p[i * n + i] += 3.4445;
        std::vector<double> y(r * c);
        for (size_t i = 0; i < r; i++)
            for (size_t j = 0; j < c; j++) {
                double s = 0;
                if (tall) for (size_t l = 0; l < c; l++) s += x[i * c + l] * p[l * c + j];
                else for (size_t l = 0; l < r; l++) s += p[i * r + l] * x[l * c + j];
                y[i * c + j] = s;
            }
        x = y;
    }
    return x;
}

static void muon_case(size_t batch, size_t r, size_t c, bool nesterov) {
    InputNode w({1, batch, r, c}, true);
    const size_t n = r * c;
    const auto vw = normal(batch * n, 30, 0.f, 0.1f);
    w.output->dataInject(vw.begin(), vw.end());
    const double lr = 0.02f, mu = 0.9f, wd = 0.1f;
    opt::Muon muon((float)lr, (float)mu, nullptr, (float)wd, nesterov);
    std::vector<double> want(vw.begin(), vw.end()), m(batch * n, 0.0);
    for (int step = 0; step < 2; step++) {
        const auto vg = normal(batch * n, 31 + step);
        w.output->dataInject(vg.begin(), vg.end(), true);
        muon.step(&w);
        double size = 0, err = 0, wsize = 0;
        for (size_t b = 0; b < batch; b++) {
            std::vector<double> u(n);
            for (size_t i = 0; i < n; i++) {
                double& mi = m[b * n + i];
                mi = mu * mi + vg[b * n + i];
                u[i] = nesterov ? vg[b * n + i] + mu * mi : mi;
            }
            const auto o = orthogonal(u, r, c);
            const double s = lr * std::sqrt(std::max(1.0, (double)r / c));
            for (size_t i = 0; i < n; i++) {
                double& v = want[b * n + i];
                v = (1 - lr * wd) * v - s * o[i];
                size += s * o[i] * s * o[i];
                wsize += v * v;
            }
        }
        const auto got = w.output->hostData();
        for (size_t i = 0; i < got.size(); i++) err += (got[i] - want[i]) * (got[i] - want[i]);
        // the operands' roundings in fp16, three products in each of five steps: 6e-3 of the update, as in the tests of
        // the operator; the second step begins with the first one's error
        EXPECT_TRUE(std::sqrt(err) <= (step + 1) * (6e-3 * std::sqrt(size) + 8 * U * std::sqrt(wsize)));
    }
    const auto state = muon.exportState(&w);
    EXPECT_TRUE(state.size() == 1 && worst(state[0], m) <= 8 * U * 8);
    // state goes over to another optimizer bit for bit
    InputNode w2({1, batch, r, c}, true);
    const auto now = w.output->hostData(), g = w.output->hostGrad();
    w2.output->dataInject(now.begin(), now.end());
    w2.output->dataInject(g.begin(), g.end(), true);
    opt::Muon other((float)lr, (float)mu, nullptr, (float)wd, nesterov);
    other.importState(&w2, state);
    muon.step(&w);
    other.step(&w2);
    EXPECT_TRUE(w.output->hostData() == w2.output->hostData());
    EXPECT_THROW(other.importState(&w2, {std::vector<float>(3)}), std::runtime_error);
}

static void test_muon() {
    muon_case(1, 64, 96, true);
    muon_case(1, 130, 64, false);
    muon_case(3, 65, 70, true);
}

static void test_muon_others() {
    InputNode bias({1, 1, 40, 1}, true), bias2({1, 1, 40, 1}, true), w({1, 1, 64, 64}, true);
    const auto v = normal(40, 40), g = normal(40, 41);
    for (InputNode* n : {&bias, &bias2}) {
        n->output->dataInject(v.begin(), v.end());
        n->output->dataInject(g.begin(), g.end(), true);
    }
    // a parameter that is no matrix goes to the other optimizer, slices too; without one it is refused
    opt::Adam adam(0.01f, 0.9f, 0.999f), alone(0.01f, 0.9f, 0.999f);
    opt::Muon muon(0.02f, 0.95f, &adam);
    muon.step(&bias);
    alone.step(&bias2);
    EXPECT_TRUE(bias.output->hostData() == bias2.output->hostData());
    EXPECT_TRUE(muon.counter() == 1 && muon.exportState(&bias) == alone.exportState(&bias2));
    muon.setSlice(&bias, 10, 20);
    alone.setSlice(&bias2, 10, 20);
    muon.step(&bias);
    alone.step(&bias2);
    EXPECT_TRUE(bias.output->hostData() == bias2.output->hostData());
    muon.setSlice(&bias, 0, 0);
    alone.setSlice(&bias2, 0, 0);
    muon.step(&bias);
    alone.step(&bias2);
    EXPECT_TRUE(bias.output->hostData() == bias2.output->hostData());
    opt::Muon bare(0.02f, 0.95f);
    EXPECT_THROW(bare.step(&bias), std::invalid_argument);
    EXPECT_TRUE(bare.exportState(&bias).empty());
    // a slice of a matrix has no singular values of its own
    w.output->fill(0.f);
    muon.setSlice(&w, 0, 64);
    EXPECT_THROW(muon.step(&w), std::runtime_error);
    // zeros stay zeros
    muon.setSlice(&w, 0, 0);
    w.output->zeroGrad();
    muon.step(&w);
    EXPECT_TRUE(w.output->hostData() == std::vector<float>(64 * 64, 0.f));
}

// A model of linear layers and norms, trained with Muon and Adam, saved in between and resumed bit for bit.
static void test_training_resumes() {
    const char* path = "/tmp/nz_token_tests_graph.json";
    NormModel m(16);
    opt::Adam adam(0.001f, 0.9f, 0.999f), adam2(0.001f, 0.9f, 0.999f);
    opt::Muon muon(0.02f, 0.95f, &adam, 0.01f), muon2(0.02f, 0.95f, &adam2, 0.01f);
    const auto before = m.parameters()[0]->output->hostData();
    run_step(m, &muon);
    EXPECT_TRUE(before != m.parameters()[0]->output->hostData());
    m.forward();
    m.backward();
    m.graph().save(path, &muon);
    graph::ComputeGraph g;
    g.load(path, &muon2);
    EXPECT_TRUE(muon2.counter() == muon.counter() && g.getNodes().size() == m.graph().getNodes().size());
    m.update(&muon);
    g.update(&muon2);
    const auto &a = m.graph().getNodes(), &b = g.getNodes();
    size_t norms = 0;
    for (size_t i = 0; i < a.size() && i < b.size(); i++) {
        EXPECT_TRUE(a[i]->type == b[i]->type && a[i]->attributes() == b[i]->attributes());
        norms += b[i]->type == "LayerNorm";
        if (a[i]->inputs.empty()) EXPECT_TRUE(a[i]->output->hostData() == b[i]->output->hostData());
    }
    EXPECT_TRUE(norms == 2);
    m.forward();
    g.forward();
    EXPECT_TRUE(m.out->output->hostData() == g.getOutputs().at(0)->inputs[0]->output->hostData());
    remove(path);
}

int main() {
    const struct { const char* name; void (*fn)(); } tests[] = {
        {"oracle", test_oracle}, {"layer_norm", test_layer_norm}, {"layer_norm_refusals", test_layer_norm_refusals}, {"model_of_norms", test_model_of_norms},
        {"muon", test_muon}, {"muon_others", test_muon_others}, {"training_resumes", test_training_resumes},
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
