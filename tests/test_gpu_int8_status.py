"""The 8-bit operators' status word (ZipNeRFCudaBackend.int8_status) at a device's first use, which a process has once: each
test runs a program of its own."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PACKAGE = Path(__file__).resolve().parent.parent / 'fused-zipnerf_b200'

PROLOGUE = f'''
import sys
sys.path.insert(0, {str(PACKAGE)!r})
import torch
import ZipNeRFCudaBackend as backend
device = torch.device('cuda:0')
# what an allocation finds if nothing clears it
dirt = [torch.full((128,), 7, dtype=torch.int32, device=device) for _ in range(64)]
torch.cuda.synchronize()
del dirt
'''

CAPTURE = '''
codes = torch.ones(40, 32, dtype=torch.int8, device=device)
scales = torch.ones(40, device=device)
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    out = backend.int8_linear(codes, scales, codes, scales)
status = backend.int8_status(device)
assert status.item() == 0, 'not cleared before the first replay'
status.fill_(1)  # as a kernel whose wait ran out
torch.cuda.synchronize()
graph.replay()
torch.cuda.synchronize()
assert status.item() == 1, 'a replay cleared the status'
assert (out == 32).all()
del graph
print('done')
'''

STREAMS = '''
late, other = torch.cuda.Stream(), torch.cuda.Stream()
x = torch.ones(4096, 4096, device=device)
torch.cuda.synchronize()
with torch.cuda.stream(late):
    for _ in range(200):
        x = x @ x
    status = backend.int8_status(device)
with torch.cuda.stream(other):
    assert status.item() == 0, 'not cleared before another stream reads it'
    status.fill_(1)  # as a kernel whose wait ran out
torch.cuda.synchronize()
assert status.item() == 1, 'the first use cleared what another stream reported'
print('done')
'''


@pytest.mark.parametrize('program', [CAPTURE, STREAMS], ids=['capture', 'streams'])
def test_the_status_at_its_first_use(program):
    run = subprocess.run([sys.executable, '-c', PROLOGUE + program], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.split()[-1] == 'done', run.stderr[-2000:]
