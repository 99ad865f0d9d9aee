// Drives layer normalisation, rotary positions and attention, forward and backward, through the C++ classes of
// distconv_b200.hpp on one rank and checks every result against plain loops in double precision.
//
// usage: shim_attention_check   (prints "shim_attention_check OK" and exits 0)
#include "distconv_b200.hpp"

#include <cmath>
#include <cstdio>
#include <vector>

using namespace distconv;

namespace
{
constexpr int W = 7, H = 5, N = 2, HEADS = 2, KV = 1, HD = 8, C = HEADS * HD, S = W * H;
constexpr double EPS = 1e-5;
typedef std::vector<double> Vec;

float synth(int i, int salt)
{
    return std::sin(0.37f * (float) (i + 1) * (float) (salt + 2)) + 0.1f * (float) salt;
}

struct Field
{
    tensor::Tensor<float> t;
    Field(int channels, int salt)
        : t(tensor::Shape({W, H, channels, N}), tensor::LocaleMPI(0, 1, nullptr),
            tensor::Distribution::make_localized_distribution(4))
    {
        t.allocate();
        std::vector<float> v((size_t) N * channels * S);
        for (size_t i = 0; i < v.size(); ++i)
            v[i] = synth((int) i, salt);
        cudaMemcpy(t.get_buffer(), v.data(), v.size() * sizeof(float), cudaMemcpyHostToDevice);
    }
    Vec host()
    {
        std::vector<float> v((size_t) t.get_local_size());
        cudaMemcpy(v.data(), t.get_buffer(), v.size() * sizeof(float), cudaMemcpyDeviceToHost);
        return Vec(v.begin(), v.end());
    }
};

std::vector<float> device_floats(const float* p, size_t n)
{
    std::vector<float> v(n);
    cudaMemcpy(v.data(), p, n * sizeof(float), cudaMemcpyDeviceToHost);
    return v;
}

int failures = 0;
void check(const char* name, const Vec& got, const Vec& want)
{
    double top = 0, off = 0;
    for (size_t i = 0; i < want.size(); ++i)
    {
        top = std::max(top, std::fabs(want[i]));
        off = std::max(off, std::fabs(got[i] - want[i]));
    }
    // sums of at most 70 fp32 products, a handful of them in a row
    if (!(off <= 1e-5 * top) || got.size() != want.size())
    {
        std::printf("%s: off by %g of %g\n", name, off, top);
        ++failures;
    }
}

size_t at(int n, int c, int s, int channels)
{
    return ((size_t) n * channels + c) * S + s;
}
} // namespace

int main()
{
    tensor::LocaleMPI loc(0, 1, nullptr);
    BackendDNNLib be(loc, 0);

    { // layer normalisation
        Field x(C, 1), y(C, 0), dy(C, 2), dx(C, 0);
        float *mem, *scale, *bias, *mean, *inv, *dw, *db;
        cudaMalloc(reinterpret_cast<void**>(&mem), sizeof(float) * (4 * C + 2 * N * S));
        scale = mem, bias = scale + C, dw = bias + C, db = dw + C, mean = db + C, inv = mean + N * S;
        std::vector<float> wb(2 * C);
        for (int i = 0; i < 2 * C; ++i)
            wb[i] = 1.f + 0.3f * synth(i, 3);
        cudaMemcpy(scale, wb.data(), sizeof(float) * 2 * C, cudaMemcpyHostToDevice);
        LayerNormalization ln(be, 4, (float) EPS);
        ln.forward(x.t, scale, bias, y.t, mean, inv);
        ln.backward(x.t, dy.t, mean, inv, scale, dw, db, dx.t);
        Field alone(C, 0); // without the gradients of scale and bias
        ln.backward(x.t, dy.t, mean, inv, scale, nullptr, nullptr, alone.t);
        be.wait();
        if (alone.host() != dx.host())
        {
            std::printf("layer norm: d_input depends on what else is wanted\n");
            return 1;
        }
        const Vec vx = x.host(), vd = dy.host();
        Vec ry(vx.size()), rx(vx.size()), rw(C, 0.), rb(C, 0.);
        for (int n = 0; n < N; ++n)
            for (int s = 0; s < S; ++s)
            {
                double m = 0, v = 0, a = 0, b = 0;
                for (int c = 0; c < C; ++c)
                    m += vx[at(n, c, s, C)] / C;
                for (int c = 0; c < C; ++c)
                    v += std::pow(vx[at(n, c, s, C)] - m, 2) / C;
                const double r = 1 / std::sqrt(v + EPS);
                for (int c = 0; c < C; ++c)
                {
                    const double u = (vx[at(n, c, s, C)] - m) * r, d = vd[at(n, c, s, C)];
                    ry[at(n, c, s, C)] = u * wb[c] + wb[C + c];
                    a += d * wb[c] / C, b += d * wb[c] * u / C;
                    rw[c] += d * u, rb[c] += d;
                }
                for (int c = 0; c < C; ++c)
                {
                    const double u = (vx[at(n, c, s, C)] - m) * r;
                    rx[at(n, c, s, C)] = r * (vd[at(n, c, s, C)] * wb[c] - a - u * b);
                }
            }
        check("norm y", y.host(), ry);
        check("norm dx", dx.host(), rx);
        const auto gw = device_floats(dw, C), gb = device_floats(db, C);
        check("norm dscale", Vec(gw.begin(), gw.end()), rw);
        check("norm dbias", Vec(gb.begin(), gb.end()), rb);
        cudaFree(mem);
    }

    { // rotary positions: there and back, and against the definition
        Field x(C, 4), y(C, 0), z(C, 0);
        RotaryPositions rot(be, 4);
        rot.setup(x.t, HD, {4, 4}, HEADS, 100.0);
        rot.forward(x.t, y.t);
        rot.backward(y.t, z.t);
        be.wait();
        const Vec v = x.host();
        Vec r = v;
        for (int n = 0; n < N; ++n)
            for (int h = 0; h < HEADS; ++h)
                for (int s = 0; s < S; ++s)
                    for (int axis = 0; axis < 2; ++axis) // H, then W
                        for (int j = 0; j < 2; ++j)
                        {
                            const double t = (axis == 0 ? s / W : s % W) * std::pow(100.0, -2.0 * j / 4);
                            const size_t p = at(n, h * HD + 4 * axis + j, s, C), q = at(n, h * HD + 4 * axis + j + 2, s, C);
                            r[p] = v[p] * std::cos(t) - v[q] * std::sin(t);
                            r[q] = v[p] * std::sin(t) + v[q] * std::cos(t);
                        }
        check("rotary", y.host(), r);
        check("rotary back", z.host(), v);
    }

    { // attention
        Field q(C, 5), k(KV * HD, 6), v(KV * HD, 7), o(C, 0), d_o(C, 8), dq(C, 0), dk(KV * HD, 0), dv(KV * HD, 0);
        float* lse;
        cudaMalloc(reinterpret_cast<void**>(&lse), sizeof(float) * N * HEADS * S);
        Attention attention(be, 4, HEADS, KV, 0.f, true);
        attention.forward(q.t, k.t, v.t, o.t, lse);
        attention.backward(q.t, k.t, v.t, o.t, lse, d_o.t, dq.t, dk.t, dv.t);
        be.wait();
        const Vec Q = q.host(), K = k.host(), V = v.host(), G = d_o.host();
        Vec O(Q.size(), 0.), DQ(Q.size(), 0.), DK(K.size(), 0.), DV(V.size(), 0.);
        const double scale = 1 / std::sqrt((double) HD);
        for (int n = 0; n < N; ++n)
            for (int h = 0; h < HEADS; ++h)
                for (int i = 0; i < S; ++i)
                {
                    Vec p(i + 1), dp(i + 1, 0.);
                    double top = -1e300, sum = 0, delta = 0;
                    for (int j = 0; j <= i; ++j)
                    {
                        double s = 0;
                        for (int c = 0; c < HD; ++c)
                            s += Q[at(n, h * HD + c, i, C)] * K[at(n, c, j, HD)];
                        p[j] = scale * s;
                        top = std::max(top, p[j]);
                    }
                    for (int j = 0; j <= i; ++j)
                        sum += p[j] = std::exp(p[j] - top);
                    for (int j = 0; j <= i; ++j)
                    {
                        p[j] /= sum;
                        for (int c = 0; c < HD; ++c)
                        {
                            O[at(n, h * HD + c, i, C)] += p[j] * V[at(n, c, j, HD)];
                            dp[j] += G[at(n, h * HD + c, i, C)] * V[at(n, c, j, HD)];
                            DV[at(n, c, j, HD)] += p[j] * G[at(n, h * HD + c, i, C)];
                        }
                        delta += p[j] * dp[j];
                    }
                    for (int j = 0; j <= i; ++j)
                        for (int c = 0; c < HD; ++c)
                        {
                            const double ds = scale * p[j] * (dp[j] - delta);
                            DQ[at(n, h * HD + c, i, C)] += ds * K[at(n, c, j, HD)];
                            DK[at(n, c, j, HD)] += ds * Q[at(n, h * HD + c, i, C)];
                        }
                }
        check("attention o", o.host(), O);
        check("attention dq", dq.host(), DQ);
        check("attention dk", dk.host(), DK);
        check("attention dv", dv.host(), DV);
        cudaFree(lse);
    }
    if (failures)
        return 1;
    std::printf("shim_attention_check OK\n");
    return 0;
}
