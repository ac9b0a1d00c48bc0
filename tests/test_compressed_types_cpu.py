"""The C++ header refuses views of other element types at compile time in the operators
on compressed data, whose calls name no type of their own."""
import concurrent.futures as cf
import os
import subprocess


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
#include <alpakann_b200/onHost.hpp>
namespace b200 = alpaka::nn::b200;
namespace nn = alpaka::nn::onHost::nn;
template <typename T, std::size_t R> b200::View<T, R> view();
void calls(b200::Queue& queue) {{
    int const exec = 0;
    auto q = view<{q}, 4>(), out = view<{q}, 4>();
    auto x = view<{x}, 4>();
    auto kc = view<int8_t, 4>();
    auto vc = view<{vc}, 4>();
    auto s = view<{s}, 3>();
    auto ko = view<float, 4>();
    auto lengths = view<{lengths}, 1>();
    auto positions = view<{positions}, 1>();
    auto in = view<{input}, 2>(), res = view<{res}, 2>(), y = view<float, 2>(), w = view<{weight}, 2>();
    auto bias = view<{bias}, 1>();
    auto packed = view<uint32_t, 2>();
    auto ws = view<float, 2>();
    auto rot = view<{rot}, 4>();
    auto f = view<double, 1>();
    nn::rotary<float>(queue, exec, rot, rot, positions, f, rot, rot);
    nn::kvCacheAppendQ8(queue, exec, x, x, kc, vc, s, s, positions, 16u, &lengths);
    nn::kvCacheAppendQ8(queue, exec, x, x, kc, vc, s, s, positions, 16u);
    nn::kvCacheReadQ8(queue, exec, kc, vc, s, s, ko, ko, 16u, &lengths);
    nn::attentionDecodeQ8(queue, exec, q, kc, vc, s, s, out, 16u, nullptr, 0.1f);
    nn::attentionDecodeQ8(queue, exec, q, kc, vc, s, s, out, 16u, &lengths, 0.1f);
    nn::packWeightQ4(queue, exec, w, packed, ws, 32u);
    nn::linearQ4(queue, exec, in, packed, ws, y, 32u, &bias, nn::Activation::silu, &res);
    nn::linearQ4(queue, exec, in, packed, ws, y, 32u);
}}
"""
TYPES = {"q": "float", "x": "float", "vc": "int8_t", "s": "float", "lengths": "int32_t", "positions": "int32_t",
         "input": "float", "res": "float", "weight": "float", "bias": "float", "rot": "float"}
WRONG = [("q", "double", "rows and scales are float"), ("x", "double", "rows and scales are float"),
         ("vc", "int32_t", "the caches are int8"), ("s", "double", "rows and scales are float"),
         ("lengths", "int64_t", "an optional view holds"), ("positions", "int64_t", "positions are int32"),
         ("input", "double", "input, scales and output are float"), ("res", "double", "an optional view holds"),
         ("weight", "double", "weight and scales are float"), ("bias", "double", "an optional view holds"),
         ("rot", "double", "of the named type")]


def compiled(types):
    r = subprocess.run(["g++", "-std=c++20", "-fsyntax-only", "-x", "c++", "-I", os.path.join(ROOT, "include"), "-I",
                        "/usr/local/cuda/include", "-"], input=PROGRAM.format(**types), capture_output=True, text=True)
    return r.returncode, r.stderr


def test_types_are_checked_at_compile_time():
    cases = [TYPES, dict(TYPES, lengths="uint32_t", positions="uint32_t")] + [dict(TYPES, **{k: t}) for k, t, _ in WRONG]
    with cf.ThreadPoolExecutor(4) as ex:
        results = list(ex.map(compiled, cases))
    for rc, err in results[:2]:
        assert rc == 0, err
    for (what, t, message), (rc, err) in zip(WRONG, results[2:]):
        assert rc != 0 and message in err, f"{what} as {t}: {err}"
