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
    { // a graph captured before another set-up
        cudaStream_t stream;
        cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
        {
            BackendDNNLib on_stream(loc, stream);
            TensorF x = shard({9, 7, 8, 1}, {1, 1, 1, 1}, 0, 1), y = shard({9, 7, 8, 1}, {1, 1, 1, 1}, 0, 1),
                    z = shard({5, 3, 8, 1}, {1, 1, 1, 1}, 0, 1);
            for (TensorF* t : {&x, &y, &z})
                t->allocate();
            std::vector<float> in((size_t) x.get_local_size()), before(in.size()), after(in.size());
            for (size_t i = 0; i < in.size(); ++i)
                in[i] = (float) (i % 23) - 11.f;
            cudaMemcpy(x.get_buffer(), in.data(), in.size() * sizeof(float), cudaMemcpyHostToDevice);
            RotaryPositions rot(on_stream, 4);
            rot.setup(x, 8, {4, 4});
            rot.forward(x, y);
            on_stream.wait();
            cudaMemcpy(before.data(), y.get_buffer(), in.size() * sizeof(float), cudaMemcpyDeviceToHost);
            cudaGraph_t graph;
            cudaGraphExec_t exec;
            cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal);
            rot.forward(x, y);
            cudaStreamEndCapture(stream, &graph);
            cudaGraphInstantiate(&exec, graph, 0);
            rot.setup(z, 8, {2, 6}, -1, 10.0);
            rot.forward(z, z);
            on_stream.wait();
            cudaMemset(y.get_buffer(), 0, in.size() * sizeof(float));
            cudaDeviceSynchronize();
            cudaGraphLaunch(exec, stream);
            on_stream.wait();
            cudaMemcpy(after.data(), y.get_buffer(), in.size() * sizeof(float), cudaMemcpyDeviceToHost);
            if (cudaGetLastError() != cudaSuccess || after != before)
                std::printf("rotary positions: a graph lost its tables\n"), ++failures;
            cudaGraphExecDestroy(exec);
            cudaGraphDestroy(graph);
        }
        cudaStreamDestroy(stream);
    }
    { // a layer's workspace: what it has grown out of stays
        internal::Workspace ws;
        void *none = ws.get(0), *small = ws.get(1000), *again = ws.get(500), *large = ws.get(1 << 20), *back = ws.get(1000);
        if (none != nullptr || again != small || large == small || back != large || cudaMemset(small, 1, 1000) != cudaSuccess
            || cudaMemset(large, 1, 1 << 20) != cudaSuccess)
            std::printf("workspace: other blocks than asked for\n"), ++failures;
    }
    if (failures)
        return 1;
    std::printf("shim_layouts_check OK\n");
    return 0;
}
