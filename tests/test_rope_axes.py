"""How ``ops.rope_store`` deals frequencies round the axes, by the rule as it is written down: frequency ``j`` to axis
``j mod axes`` as long as that has any left, else to the first.  Sections that come out of the rule are taken,
others refused."""
import itertools

import pytest

from tq4_decode import ops


def dealt(sections, half):
    left, axes = list(sections), []
    for j in range(half):
        a = j % len(sections)
        if a == 0 or left[a] == 0:
            a = 0
        left[a] -= 1
        axes.append(a)
    return axes, all(n == 0 for n in left)


@pytest.mark.parametrize("half", [8, 16, 24, 32, 40, 48, 56, 64])
@pytest.mark.parametrize("axes", [2, 3])
def test_dealt_by_the_rule(half, axes):
    for rest in itertools.product(range(half + 1), repeat=axes - 1):
        sections = (half - sum(rest), *rest)
        if sections[0] < 0:
            continue
        want, taken = dealt(sections, half)
        if taken:
            assert list(ops._axis_of(sections, True, half)) == want, sections
        else:
            with pytest.raises(RuntimeError, match="in turn"):
                ops._axis_of(sections, True, half)


@pytest.mark.parametrize("sections", [(11, 11, 10), (3, 3, 2), (22, 21, 21), (6, 6, 6, 6), (13, 13, 12, 12)])
def test_even_deals(sections):
    """The axes in strict turn, also where their number does not divide the frequencies."""
    half = sum(sections)
    assert list(ops._axis_of(sections, True, half)) == [j % len(sections) for j in range(half)]
