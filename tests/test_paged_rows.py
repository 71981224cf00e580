"""Where an append's tokens go when cu_q is wrong: a token that its sequence does
not have is written nowhere (csrc/sa_paged_plan.h's append_row, enumerated)."""
from test_paged_plan import ask  # noqa: F401 (the fixture)


def test_tokens_that_the_sequence_does_not_have(ask):  # noqa: F811
    # len n t max_pages page_log2 pos0 n_pos; a range that runs backwards has n < 0
    got = ask(["row 10 4 3 8 4 0 100", "row 10 4 4 8 4 0 100", "row 10 4 7 8 4 0 100", "row 10 -1 2 8 4 0 100",
               "row 10 0 0 8 4 0 100", "row 10 4 -1 8 4 0 100", "row 10 -5 -3 8 4 0 100"])
    assert got == [[9], [-1], [-1], [-1], [-1], [-1], [-1]]


def test_every_written_row_is_one_of_the_sequence(ask):  # noqa: F811
    cases = [(length, n, t) for length in (0, 1, 16, 33) for n in range(-3, 6) for t in range(-3, 8)]
    for (length, n, t), (row,) in zip(cases, ask(f"row {a} {b} {c} 4 4 0 1000" for a, b, c in cases)):
        right = 0 <= t < n and length - n + t >= 0
        assert row == (length - n + t if right else -1) and (row == -1 or row < length)
