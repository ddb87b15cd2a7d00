"""Refusals of layer norm, dropout and the residual step that need no device."""
import pytest
import torch


def test_make_fx_is_refused():
    """make_fx would record the allocation of a result and not the kernel that fills it."""
    import siv.backend as sb
    from siv import ops, rng
    from torch.fx.experimental.proxy_tensor import make_fx
    sb.set_backend(None)
    k = rng.PhiloxKeep(1, 2)
    for call in (lambda x: ops.layer_norm(x), lambda x: ops.dropout(x, k, 0.5), lambda x: ops.act_dropout(x, 0.0, k, 0.5),
                 lambda x: ops.add_layer_norm(x, x)):
        for mode in ("real", "fake", "symbolic"):
            with pytest.raises(Exception, match="make_fx"):
                make_fx(call, tracing_mode=mode)(torch.zeros(2, 8))
