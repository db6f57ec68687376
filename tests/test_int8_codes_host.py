"""The arithmetic by which the 8-bit row operators turn values into codes (csrc/fz_int8_rows.cu: the product with the scale's
reciprocal in two floats), restated on the host: at the half steps, where the code changes, it gives the code of the fp32
quotient. No GPU needed."""
from __future__ import annotations

import subprocess

PROGRAM = r'''
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
static float from_bits(uint32_t u) { float v; std::memcpy(&v, &u, 4); return v; }
static uint32_t bits(float v) { uint32_t u; std::memcpy(&u, &v, 4); return u; }
int main() {
    long checked = 0;
    // one exponent stands for all: the products scale by powers of two
    for (uint32_t significand = 0; significand < (1u << 23); significand += significand % 8192 < 64 ? 1 : 113) {
        const float scale = from_bits(127u << 23 | significand);
        const float high = static_cast<float>(1.0 / static_cast<double>(scale));
        const float error = fmaf(-high, scale, 1.0f), low = high * fmaf(error, error, error);
        for (int k = 0; k < 127; k++) {
            const float half = static_cast<float>((k + 0.5) * static_cast<double>(scale));
            for (int step = -2; step <= 2; step++) {
                const float v = from_bits(bits(half) + step), quotient = v / scale;
                checked++;
                if (std::nearbyint(fmaf(v, high, v * low)) != std::nearbyint(quotient)) {
                    std::printf("scale %a value %a\n", scale, v);
                    return 1;
                }
            }
        }
    }
    std::printf("%ld values\n", checked);
    return 0;
}
'''


def test_codes_at_the_half_steps(tmp_path):
    source, binary = tmp_path / 'codes.cpp', tmp_path / 'codes'
    source.write_text(PROGRAM)
    subprocess.run(['g++', '-std=c++17', '-O2', '-ffp-contract=off', str(source), '-o', str(binary)], check=True, timeout=120)
    run = subprocess.run([str(binary)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout
    assert int(run.stdout.split()[0]) > 10_000_000
