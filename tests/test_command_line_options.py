"""Options of the command line that cannot be used end it with status 2 and the reason, before a model is looked for.  No GPU."""

import pytest


@pytest.mark.parametrize("options,why", [
    (["--mode", "temperature", "--temperature", "0"], "temperature"), (["--mode", "top_p", "--top-p", "1.5"], "top_p"),
    (["--presence-penalty", "nan"], "presence_penalty"), (["--frequency-penalty", "1e31"], "frequency_penalty"),
    (["--repetition-penalty", "0"], "repetition_penalty"), (["--logit-bias", "7"], "logit-bias"), (["--logit-bias", "7:x"], "logit-bias"),
    (["--logit-bias", "7:1:2"], "logit-bias"), (["--logit-bias=-1:2"], "logit_bias"), (["--logit-bias", "7:inf"], "finite")])
def test_refused(options, why, capsys):
    from inf_engine_b200.cli.generate import main
    assert main(["--model-dir", "/nowhere", "--prompt-ids", "1,2", *options]) == 2
    assert why in capsys.readouterr().err
