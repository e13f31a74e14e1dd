"""Calls of ``ops.rope_store`` at the edges of what it takes: sections that deal the frequencies evenly round the axes."""
import pytest

from test_gpu_rope_store import build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rot,sections", [(64, (11, 11, 10)), (16, (3, 3, 2)), (128, (22, 21, 21)), (96, (12, 12, 12, 12))])
@pytest.mark.parametrize("neox", [True, False])
def test_evenly_dealt_axes(dev, rot, sections, neox):
    for preset in ("4bit", "k8v4"):
        check(dev, build(21, 90, 4, 2, preset, rot=rot, neox=neox, sections=sections, in_turn=True))
