"""GPU: the status word of the paged kernels, on other streams and whoever makes the first call."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from paged_util import make_batch

pytestmark = pytest.mark.gpu


def _append(cuda, bad):
    """An append of one row; `bad`: its page is outside the pool."""
    from omlx_exl3_b200 import paged_qkv_post
    b = make_batch([1], [3], 1, 64, 16, torch.float16, cuda)
    table = b["table"] + (99 if bad else 0)
    y = torch.zeros((1, 3 * 64), dtype=torch.float16, device=cuda)
    angle = torch.zeros((8, 32), device=cuda)
    return lambda: paged_qkv_post(*y.split(64, 1), None, None, 1e-6, angle.cos(), angle.sin(), b["kp"], b["vp"], table, b["cu"], b["lens"])


def test_a_bit_set_on_another_stream_is_seen(cuda):
    """The check waits for every stream of the device, not its own alone."""
    from omlx_exl3_b200 import check_paged_status
    from omlx_exl3_b200.paged import paged_status
    call = _append(cuda, True)
    call()
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)
    check_paged_status(cuda)
    side = torch.cuda.Stream()
    for look in (check_paged_status, paged_status):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
            call()
        if look is paged_status:
            assert paged_status(cuda) == 8 and paged_status(cuda) == 8
        with pytest.raises(RuntimeError, match="outside its range"):
            check_paged_status(cuda)
    assert paged_status(cuda) == 0


FIRST = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
from test_paged_status_gpu import _append
from omlx_exl3_b200 import check_paged_status
from omlx_exl3_b200._lib import torch_calls
cuda = torch.device("cuda:0")
torch_calls()
call = _append(cuda, True)
torch.cuda.synchronize()
{first}
torch.cuda.synchronize()
for word in ("outside its range", None):
    try:
        check_paged_status(cuda)
    except RuntimeError as e:
        assert word and word in str(e), e
    else:
        assert word is None
print("fine")
"""

INFERENCE = """
with torch.inference_mode():
    call()
"""

# the first call's stream is busy: the fill of the word must not come after another stream's bit
BUSY = """
late, soon = torch.cuda.Stream(), torch.cuda.Stream()
good = _append(cuda, False)
for s in (late, soon):
    with torch.cuda.stream(s):
        torch.zeros(4, device=cuda)                          # the stream has memory: asking for some may wait for the device
torch.cuda.synchronize()
with torch.cuda.stream(late):
    torch.cuda._sleep(2_000_000_000)
    good()
with torch.cuda.stream(soon):
    call()
"""


@pytest.mark.parametrize("first", [INFERENCE, BUSY])
def test_first_call(cuda, first):
    """A process whose first paged call is made under inference mode, or on a stream with work ahead of it."""
    here = Path(__file__).resolve().parent
    # modules loaded as the process starts: loading one at its first launch may wait for the device
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=str(here.parent), tests=str(here), first=first)], capture_output=True,
                       text=True, timeout=300, env={**os.environ, "CUDA_MODULE_LOADING": "EAGER"})
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
