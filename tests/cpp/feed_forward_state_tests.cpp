// What a FeedForwardBlock keeps between its calls, and which calls it refuses for the lack of it.
#include <cmath>

#include "DotCompute/FeedForward.hpp"
#include "test_framework.hpp"

using namespace DotCompute;
using DotCompute::Algorithms::Activation;
using DotCompute::Algorithms::AdamWOptions;
using DotCompute::Algorithms::FeedForwardBlock;
using DotCompute::Algorithms::Matrix;

namespace {

std::shared_ptr<Backends::Hip::HipAccelerator> Device() {
  auto acc = Backends::Hip::TryCreateAccelerator();
  CHECK(acc != nullptr);
  return acc;
}

}  // namespace

// More than 2^23 outputs are refused by the first product, after the norm has been enqueued.
TEST_GPU(feed_forward_block_keeps_nothing_of_a_forward_that_throws) {
  auto acc = Device();
  FeedForwardBlock block(1, (1 << 23) + 1, Activation::Relu, *acc);
  CHECK_THROWS(NotSupportedException, block.Forward(Matrix(2, 1)));
  CHECK_THROWS(InvalidOperationException, block.Backward(Matrix(2, 1)));
}

// Gradients are those of the network that Forward ran: new values of the parameters ask for a new Forward.
TEST_GPU(feed_forward_block_refuses_a_backward_of_other_parameters) {
  auto acc = Device();
  const Matrix x(2, 3, {1, -2, 3, 0.5f, 2, -1});
  for (bool set : {false, true}) {
    FeedForwardBlock block(3, 4, Activation::Silu, *acc);
    block.Forward(x);
    block.Backward(x);
    block.Backward(x);  // (the same network: as often as one likes)
    if (set) block.Set(FeedForwardBlock::W1, std::vector<float>(12, 0.5f));
    else block.Step(AdamWOptions());
    CHECK_THROWS(InvalidOperationException, block.Backward(x));
    block.Forward(x);
    CHECK(block.Backward(x).Rows() == 2);
  }
}

// The gradients stay readable after the step that took them, which is taken once.
TEST_GPU(feed_forward_block_keeps_gradients_past_a_step) {
  auto acc = Device();
  const Matrix x(2, 3, {1, -2, 3, 0.5f, 2, -1});
  FeedForwardBlock block(3, 4, Activation::Silu, *acc);
  block.Forward(x);
  block.Backward(x);
  const auto before = block.Gradient(FeedForwardBlock::B2);
  CHECK(before == (std::vector<float>{1.5f, 0.0f, 2.0f}));  // (the sums of dy's columns)
  block.Step(AdamWOptions());
  CHECK(block.Gradient(FeedForwardBlock::B2) == before);
  CHECK_THROWS(InvalidOperationException, block.Step(AdamWOptions()));
}

// Sums over more than 2^23 rows are refused.
TEST_GPU(feed_forward_block_keeps_no_gradients_of_a_backward_that_throws) {
  auto acc = Device();
  FeedForwardBlock block(1, 1, Activation::None, *acc);
  block.Forward(Matrix(2, 1));
  block.Backward(Matrix(2, 1));
  const Matrix tall((1 << 23) + 1, 1);
  block.Forward(tall);
  CHECK_THROWS(NotSupportedException, block.Backward(tall));
  CHECK_THROWS(InvalidOperationException, block.Gradient(FeedForwardBlock::W2));
  CHECK_THROWS(InvalidOperationException, block.Step(AdamWOptions()));
}
