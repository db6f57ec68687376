"""What the int8 weight gradient's off-grid path reads of its gradients (csrc/fz_grad_words.h), restated over all layouts on
the host: every element of every word lies in the tensor. No GPU needed."""
from __future__ import annotations

import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / 'fused-zipnerf_b200' / 'csrc'

# the loads of one call, for a tensor whose memory is exactly the elements [0, (n - 1) stride + out) behind a base that may
# lie in the middle of a 32-bit word: the CTAs' columns, the workers' rows and the lanes' words as the kernel has them
PROGRAM = r'''
#include "fz_grad_words.h"
#include <algorithm>
#include <cstdio>
using namespace zf::int8_weight_grad;
int main() {
    constexpr int kRows = 64, kTeam = 8;
    long checked = 0;
    for (int n : {1, 63, 64, 65, 127, 128, 129, 130, 140, 191, 192, 193, 256, 257, 4133})
        for (int out : {1, 2, 3, 5, 7, 9, 61, 63, 64, 65, 127, 128, 129, 130, 131, 255, 256, 257, 300, 383, 384, 385})
            for (int pad : {0, 1, 2, 3})
                for (int base : {0, 1}) {
                    const long stride = out + pad, end = (n - 1) * stride + out;
                    for (int tile = 0; 256 * tile < out; tile++)
                        for (int rank = 0; rank < 2; rank++) {
                            const int out0 = 256 * tile + 128 * rank, columns = std::max(0, std::min(128, out - out0));
                            for (int row0 = 0; row0 < n; row0 += kRows) {
                                if (!whole_words(row0, kRows, n)) continue;  // element by element, each behind its own check
                                for (int w = 0; w < kTeam; w++) {
                                    const int odd = static_cast<int>((base + w * stride + out0) & 1);
                                    for (int r = 0; r < kRows / kTeam; r++)
                                        for (int word = 0; word <= 64; word++) {
                                            if (!word_needed(word, odd, columns)) continue;
                                            const long first = (row0 + w + kTeam * r) * stride + out0 + word_column(word, odd);
                                            checked++;
                                            if (first < 0 || first + 1 >= end || ((base + first) & 1)) {
                                                std::printf("n %d out %d stride %ld base %d: word at %ld of %ld\n", n, out, stride, base, first, end);
                                                return 1;
                                            }
                                        }
                                }
                            }
                        }
                }
    std::printf("%ld words\n", checked);
    return 0;
}
'''


def test_every_word_of_a_gradient_lies_in_the_tensor(tmp_path):
    source, binary = tmp_path / 'words.cpp', tmp_path / 'words'
    source.write_text(PROGRAM)
    subprocess.run(['g++', '-std=c++17', '-O2', '-I', str(CSRC), str(source), '-o', str(binary)], check=True, timeout=120)
    run = subprocess.run([str(binary)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout
    assert int(run.stdout.split()[0]) > 1_000_000
