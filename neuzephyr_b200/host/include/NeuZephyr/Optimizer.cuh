// Optimizers used by the training step (mirrors include/NeuZephyr/Optimizer.cuh,
// src/Optimizer.cu:79-102): SGD and Adam, and Muon beside them. Adam keeps the reference's quirk of one time step per
// step(Node*) call (the counter is shared by all parameters), eps 1e-6.
#pragma once
#include <memory>
#include <unordered_map>
#include <utility>
#include <vector>

#include "Nodes.cuh"

namespace nz::opt {

class Optimizer {
public:
    virtual ~Optimizer() = default;
    virtual void step(nodes::Node* input) = 0;
    // `n` step() calls the reference would have made on nodes this graph does not step
    // (activations, nodes folded into a fused node): only per-call state advances.
    virtual void skip(int n) { (void)n; }
    // ComputeGraph::update brackets its loop with these: an optimizer may collect the step() calls in
    // between and run them as one launch in endBatch() (Adam does). The default runs each step at once.
    virtual void beginBatch() {}
    virtual void endBatch() {}
    // A step between the two threw: the steps collected so far (and their counts) are forgotten, and the next one runs at once.
    virtual void dropBatch() {}
    // Throws if step(node) would be refused; `sliced`: with a slice of the node. Touches nothing. Model::update and
    // ComputeGraph::update ask for every node before they exchange a gradient or take a step.
    virtual void checkStep(nodes::Node* node, bool sliced) const { (void)node; (void)sliced; }
    // Restricts the steps of `node` to elements [offset, offset + count) of its tensor (count == 0: the
    // whole tensor again). A data-parallel run with a sharded optimizer gives every rank its own slice.
    void setSlice(nodes::Node* node, size_t offset, size_t count) {
        if (count) slices_[node] = {offset, count};
        else slices_.erase(node);
    }
    bool hasSlice(nodes::Node* node) const { return slices_.count(node) != 0; }

protected:
    std::pair<size_t, size_t> sliceOf(nodes::Node* node) const {
        auto it = slices_.find(node);
        return it == slices_.end() ? std::pair<size_t, size_t>{0, node->output->size()} : it->second;
    }
    std::unordered_map<nodes::Node*, std::pair<size_t, size_t>> slices_;

public:
    // Checkpointing (ComputeGraph::save / load): a name, the per-call counter, and per node the state
    // vectors the optimizer keeps (empty when it keeps none for that node).
    virtual const char* name() const { return "Optimizer"; }
    virtual long counter() const { return 0; }
    virtual void setCounter(long) {}
    virtual std::vector<std::vector<float>> exportState(nodes::Node*) const { return {}; }
    virtual void importState(nodes::Node*, const std::vector<std::vector<float>>&) {}

protected:
    float learning_rate = 0.f;
};

class SGD : public Optimizer {
public:
    explicit SGD(float learning_rate);
    void step(nodes::Node* input) override;
    const char* name() const override { return "SGD"; }
};

class Adam : public Optimizer {
public:
    Adam(float learning_rate, float beta1, float beta2);
    void step(nodes::Node* input) override;
    void skip(int n) override { it_ += n; }
    void beginBatch() override;
    void endBatch() override;  // one nzb_adam_multi launch over every tensor stepped since beginBatch()
    void dropBatch() override;
    const char* name() const override { return "Adam"; }
    long counter() const override { return it_; }
    void setCounter(long it) override { it_ = (int)it; }
    // {first moments, second moments} of a node, in host memory
    std::vector<std::vector<float>> exportState(nodes::Node* node) const override;
    void importState(nodes::Node* node, const std::vector<std::vector<float>>& state) override;
    // false restores "one time step per optimisation step" semantics: call nextIteration() once
    // per Model::update and every parameter uses the same t
    bool perCallTimeStep = true;
    void nextIteration() { it_shared_++; }

private:
    float beta1_, beta2_, epsilon_ = 1e-6f;
    int it_ = 0, it_shared_ = 0, it_before_batch_ = 0;
    bool batching_ = false;
    std::vector<std::pair<nodes::Node*, int>> batch_;  // (node, time step) collected between begin / endBatch
    std::unordered_map<nodes::Node*, std::unique_ptr<data::Tensor>> m_, v_;
};

// Muon (no counterpart in the reference): momentum, then the update with its singular values brought near 1 by five
// Newton-Schulz products (nzb_muon); w = (1 - lr * weight_decay) * w - lr * sqrt(max(1, outputs / inputs)) * update. It takes
// weights whose H and W are above 1, as N*C matrices: what Linear (outputs by inputs) and Conv2d (inputs by outputs) name
// as such, and what has no role, read as outputs by inputs. Biases (a convolution's {1, 1, Ho*Wo, Cout} too), norms and
// vectors go to `others`, which the caller owns and which keeps its own learning rate, counter and state.
class Muon : public Optimizer {
public:
    Muon(float learning_rate, float momentum, Optimizer* others = nullptr, float weight_decay = 0.f, bool nesterov = true);
    void step(nodes::Node* input) override;
    void skip(int n) override { if (others_) others_->skip(n); }
    void beginBatch() override { if (others_) others_->beginBatch(); }
    void endBatch() override { if (others_) others_->endBatch(); }
    void dropBatch() override { if (others_) others_->dropBatch(); }
    void checkStep(nodes::Node* node, bool sliced) const override;
    const char* name() const override { return "Muon"; }
    long counter() const override { return others_ ? others_->counter() : 0; }
    void setCounter(long it) override { if (others_) others_->setCounter(it); }
    // {momentum} of a matrix, in host memory; the state of `others` for the rest
    std::vector<std::vector<float>> exportState(nodes::Node* node) const override;
    void importState(nodes::Node* node, const std::vector<std::vector<float>>& state) override;

private:
    static bool isMatrix(nodes::Node* node);
    float mu_, weight_decay_;
    bool nesterov_;
    Optimizer* others_;
    std::unordered_map<nodes::Node*, std::unique_ptr<data::Tensor>> momentum_;
};

}  // namespace nz::opt
