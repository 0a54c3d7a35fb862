"""AdamW checks the options of each group of parameters, not only its defaults."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


def test_group_options(pkg):
    def group(**kw):
        return dict(params=[torch.zeros(8)], **kw)
    opt = pkg.AdamW([group(lr=1e-2, state_bits=8), group(weight_decay=0.0)], lr=1e-3)
    assert [g["state_bits"] for g in opt.param_groups] == [8, 32] and [g["lr"] for g in opt.param_groups] == [1e-2, 1e-3]
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(0.9, 1.0)), dict(eps=-1.0),
                dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError):
            pkg.AdamW([group(), group(**bad)])
        with pytest.raises(ValueError):
            opt.add_param_group(group(**bad))
    with pytest.raises(TypeError):
        pkg.AdamW([group(lr=torch.tensor(1e-3))])
    assert len(opt.param_groups) == 2
