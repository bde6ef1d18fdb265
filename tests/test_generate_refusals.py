"""What parallel sampling refuses before it uses the model."""

from __future__ import annotations

import pytest

from ptxgen.generate import generate


@pytest.mark.parametrize("prompts,samples,steps", [([], 2, 3), ([[1, 2], []], 2, 3),
                                                   ([[], [5]], 2, 3), ([[1]], 0, 3),
                                                   ([[1]], -1, 3), ([[1]], 2, 0)])
def test_a_prompt_a_sample_and_a_step_at_least(prompts, samples, steps) -> None:
    with pytest.raises(ValueError, match="at least one"):
        generate(None, prompts, samples, steps)
