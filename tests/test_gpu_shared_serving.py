"""Page tables, attention behind a prefix, forks, compaction and chosen pages in one run, as a server would use them."""
import pytest

torch = pytest.importorskip("torch")

from examples import shared_serving as S  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [1, 40])
def test_the_example(steps):
    """bf16 outputs: half a unit is 2^-8 of the value, P's rounding 2^-11 of sum p |v|, binary32 2^-13 of it on either side. The pages that are held
    are those of the rows that are left, full ones of a question once for all its answers."""
    questions, answers, instruction = (37, 160, 5), 3, 1000
    worst, held = S.run(steps, instruction, questions, answers)
    assert worst <= 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12
    live = [(q, a) for q in range(3) for a in range(answers)][1:-1]  # (the first answer and the last have ended, and the first question)
    page = S.PAGE
    pages = -(-instruction // page)
    for q, n in enumerate(questions):
        mine = [a for x, a in live if x == q]
        own = -(-(n + steps) // page) - n // page
        pages += (n // page if mine or q else 0) + len(mine) * own + (1 if q and n % page else 0)
    assert held == pages
