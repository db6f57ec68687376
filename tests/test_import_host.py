"""The package imports first in a process, before torch, as well as after it. No GPU needed."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parent.parent / 'fused-zipnerf_b200'


@pytest.mark.parametrize('first', ['', 'import torch; '])
@pytest.mark.parametrize('statement', ['import ZipNeRFCudaBackend', 'from ZipNeRFCudaBackend import _C', 'from ZipNeRFCudaBackend.torch_bindings import pipeline'])
def test_the_package_imports(first, statement):
    run = subprocess.run([sys.executable, '-c', f'import sys; sys.path.insert(0, {str(PACKAGE)!r}); {first}{statement}'], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
