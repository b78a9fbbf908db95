"""The largest call of q4mi_logits_process, from both sides of its limit as
far as no GPU is needed (test_gpu_logits_slices runs the largest one)."""
import os
import re

from conftest import ROOT

import q4mi

A = 1 << 20     # an aligned address that no refused call touches


def test_workgroups_stay_below_2_to_23():
    """512 threads a workgroup: 2^23 of them are 2^32 threads, one too many
    for a launch."""
    def call(rows, vocab):
        return q4mi.lib().q4mi_logits_process(A, q4mi.T_F16, vocab, rows, vocab, None, None, None,
                                              None, None, None, None, None, 0, 0, None, A, vocab)

    for rows, vocab in ((1 << 23, 1), (1 << 23, 8192), (1 << 22, 8193), (1 << 6, 1 << 30)):
        assert not call(rows, vocab)
        assert "too large" in q4mi.last_error(), q4mi.last_error()


def test_header_says_so():
    text = open(os.path.join(ROOT, "include", "q4mi.h")).read()
    text = re.sub(r"\s*\n \*\s*", " ", text)
    assert "Fewer than 2^23 workgroups of 2048 to 8192 tokens of a row" in text
