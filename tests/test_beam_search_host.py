"""Tracing hypotheses back (no GPU needed)."""
import numpy as np

from pvlc_b200 import beam, greedy


def test_hypotheses_trace_back_through_the_beams():
    tok = np.array([[5, 6], [7, 8], [9, 1]])
    par = np.array([[0, 0], [1, 0], [0, 1]])
    inf = -np.inf
    # one ended at token 3 from beam 1 of step 2 (token 8, from beam 0: token 5)
    got = beam.hypotheses(tok, par, [-0.5, inf], [3, 0], [1, 0], False, [-3.0, -4.5], 1.0)
    assert got == [(-0.5, [5, 8], greedy.EOS_TOKEN), (-1.0, [6, 7, 9], greedy.MAX_NEW_TOKENS)]
    # a done request's live beams do not count
    got = beam.hypotheses(tok, par, [-0.5, -0.75], [3, 1], [1, 0], True, [0.0, 0.0], 1.0)
    assert got == [(-0.5, [5, 8], greedy.EOS_TOKEN), (-0.75, [], greedy.EOS_TOKEN)]
    # equal scores: the ended one first; dead beams are none
    got = beam.hypotheses(tok, par, [-1.0, inf], [2, 0], [1, 0], False, [-9.0, inf], 2.0)
    assert got == [(-1.0, [6], greedy.EOS_TOKEN), (-1.0, [6, 7, 9], greedy.MAX_NEW_TOKENS)]
