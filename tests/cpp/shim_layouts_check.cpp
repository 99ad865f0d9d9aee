// Layouts and calls that LayerNormalization, RotaryPositions and Attention of distconv_b200.hpp refuse, and what has to
// stay alive behind a captured graph.  One rank; tensors of two-rank layouts are described, not allocated.
//
// usage: shim_layouts_check   (prints "shim_layouts_check OK" and exits 0)
#include "distconv_b200.hpp"

#include <cstdio>
#include <stdexcept>
#include <vector>

using namespace distconv;

namespace
{
int failures = 0;

template <class F>
void refused(const char* name, F f)
{
    try
    {
        f();
        std::printf("%s: not refused\n", name);
        ++failures;
    }
    catch (const std::invalid_argument&)
    {}
    catch (const std::exception& e)
    {
        std::printf("%s: refused for another reason: %s\n", name, e.what());
        ++failures;
    }
}

TensorF shard(const tensor::Shape& shape, const tensor::Shape& grid, int rank, int size)
{
    return TensorF(shape, tensor::LocaleMPI(rank, size, nullptr), tensor::Distribution::make_distribution(grid));
}
} // namespace

int main()
{
    tensor::LocaleMPI loc(0, 1, nullptr);
    BackendDNNLib be(loc, 0);

    { // a cell's channels on two ranks
        TensorF cut = shard({6, 4, 8, 2}, {1, 1, 2, 1}, 0, 2), whole = shard({6, 4, 4, 2}, {1, 1, 1, 1}, 0, 1);
        LayerNormalization ln(be, 4, 1e-5f);
        refused("layer norm", [&] { ln.forward(cut, nullptr, nullptr, whole); });
        refused("layer norm, output", [&] { ln.forward(whole, nullptr, nullptr, cut); });
        refused("layer norm backward",
                [&] { ln.backward(whole, cut, nullptr, nullptr, nullptr, nullptr, nullptr, whole); });
    }
    { // cells at other positions than the layer was set up for
        TensorF first = shard({12, 6, 8, 2}, {2, 1, 1, 1}, 0, 2), second = shard({12, 6, 8, 2}, {2, 1, 1, 1}, 1, 2),
                cut = shard({6, 6, 16, 2}, {1, 1, 2, 1}, 0, 2);
        RotaryPositions rot(be, 4);
        refused("rotary positions, channels", [&] { rot.setup(cut, 4, {2, 2}); });
        rot.setup(first, 4, {2, 2});
        refused("rotary positions, place", [&] { rot.forward(second, second); });
        refused("rotary positions, output", [&] { rot.backward(first, second); });
        refused("rotary positions, channels", [&] { rot.forward(cut, cut); });
    }
    if (failures)
        return 1;
    std::printf("shim_layouts_check OK\n");
    return 0;
}
