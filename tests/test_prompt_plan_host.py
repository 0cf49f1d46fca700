"""How sn_mamba2_prompt cuts prompts into segments, as far as it shows without a GPU: in the source."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "sonata_b200" / "csrc"


def test_waves_are_of_the_device_at_hand():
    """The plan counts waves over the device's SMs, not over a number written down."""
    code = re.sub(r"//[^\n]*", "", (CSRC / "mamba_prompt.cu").read_text())
    assert "sms = sm_count()" in code
    assert not re.search(r"\b(148|132|144)\b", code)
