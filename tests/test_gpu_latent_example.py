"""The example layer: a training step lowers its loss, and the prompt's and the
decoded tokens' outputs are the expanded form's over the whole sequence."""

import importlib.util
from pathlib import Path

import pytest


@pytest.mark.gpu
def test_layer_trains_and_decodes_what_the_expanded_form_says():
    path = Path(__file__).resolve().parents[1] / "examples" / "latent_layer.py"
    spec = importlib.util.spec_from_file_location("latent_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    (before, after), prompt, decoded = m.run()
    assert after < before
    # bf16: some ten roundings lie between the forms (queries, latents, keys and
    # values, probabilities, outputs), each of 2^-9 / sqrt(3) rms = 1.1e-3 of its
    # value and none amplified by more than the scores' size of about four
    assert prompt < 10 ** 0.5 * 4 * 2 ** -9 / 3 ** 0.5
    assert decoded < 10 ** 0.5 * 4 * 2 ** -9 / 3 ** 0.5
