"""How sn_mamba2_prompt cuts prompts into segments, as far as it shows without a GPU: in the workspace's size, and in the
source."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "sonata_b200" / "csrc"


@pytest.fixture(scope="module")
def L():
    from sonata_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_most_tokens(L):
    """Token counts up to the last int plan alike: the sizes go on as they were."""
    size = lambda t: L.sn_mamba2_prompt_workspace_size(t, 1, 128, 1, 128, 2)
    a, b = size(2 ** 31 - 1 - 256), size(2 ** 31 - 1)
    assert a <= b <= a * 1.001


def test_waves_are_of_the_device_at_hand():
    """The plan counts waves over the device's SMs, not over a number written down."""
    code = re.sub(r"//[^\n]*", "", (CSRC / "mamba_prompt.cu").read_text())
    assert "sms = sm_count()" in code
    assert not re.search(r"\b(148|132|144)\b", code)
