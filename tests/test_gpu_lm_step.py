"""Layer normalisation, fully connected softmax loss and Muon solver together, as a training step uses them: a chain through vl_simplenn, its
gradients against the separate layers and against differences of the loss, and the trainer's update of all its parameters."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _net(mat, rng, classes, maps=False):
    t = lambda *s: mat.from_numpy((rng.standard_normal(s) / np.sqrt(np.prod(s[:3]))).astype(np.float32))       # noqa: E731
    one = lambda k: mat.from_numpy(np.ones((k, 1), np.float32))                                               # noqa: E731
    zero = lambda *s: mat.zeros(s)                                                                            # noqa: E731
    if maps:
        layers = [dict(type="conv", weights=[t(3, 3, 3, 24), zero(1, 24)], pad=1), dict(type="layernorm", weights=[one(24), zero(24, 1)]), dict(type="relu"),
                  dict(type="pool", pool=[2, 2], stride=2), dict(type="fcsoftmaxloss", weights=[t(4, 4, 24, classes), zero(classes, 1)])]
    else:
        layers = [dict(type="layernorm", weights=[one(40), zero(40, 1)], epsilon=1e-4), dict(type="conv", weights=[t(1, 1, 40, 96), zero(1, 96)]),
                  dict(type="relu"), dict(type="layernorm", weights=[one(96), zero(96, 1)]), dict(type="fcsoftmaxloss", weights=[t(1, 1, 96, classes), None])]
    return {"layers": layers}


def _data(mat, rng, maps, n, classes):
    x = mat.from_numpy(rng.standard_normal((8, 8, 3, n) if maps else (1, 1, 40, n)).astype(np.float32))
    c = rng.integers(0, classes + 1, n).astype(np.float32)
    import torch
    return x, torch.from_numpy(c).cuda()


@pytest.mark.parametrize("maps,n,classes", [(False, 50, 333), (True, 12, 70), (False, 3, 1000)])
def test_chain_against_separate_layers_and_differences(gpu, maps, n, classes):
    from matconvnet_b200 import simplenn
    nn, mat, _ = gpu
    rng = np.random.default_rng(0)
    net = _net(mat, rng, classes, maps)
    x, c = _data(mat, rng, maps, n, classes)
    net["layers"][-1]["class"] = c
    res = simplenn.vl_simplenn(net, x, 1.0)
    last = net["layers"][-1]
    split = {"layers": net["layers"][:-1] + [dict(type="conv", weights=last["weights"]), dict(type="softmaxloss", **{"class": c})]}
    ref = simplenn.vl_simplenn(split, x, 1.0)
    rel = lambda a, b: float((a - b).norm() / b.norm().clamp(min=1e-30))                                       # noqa: E731
    assert rel(res[-1]["x"].view(-1), ref[-1]["x"].view(-1)) < 2e-6
    for i in range(len(net["layers"])):
        # both sides are within 1e-5 of the exact derivatives, layer by layer; five layers
        assert rel(res[i]["dzdx"], ref[i]["dzdx"]) < 1e-4
        for p, q in zip(res[i]["dzdw"] or [], ref[i]["dzdw"] or []):
            assert (p is None) == (q is None)
            if p is not None:
                assert rel(p.reshape(-1), q.reshape(-1)) < 1e-4
    # differences of the loss along the gradient of the last filter bank, where the loss is smooth: the second-order term is below 1% at this step
    df = res[len(net["layers"]) - 1]["dzdw"][0]
    f = last["weights"][0]
    h = 0.05 / float(df.norm())
    losses = []
    for s in (h, -h):
        f.add_(s * df)
        losses.append(float(simplenn.vl_simplenn(net, x)[-1]["x"]))
        f.sub_(s * df)
    want = float((df * df).sum())
    # the loss, of order 6, carries 2e-6 of itself; the difference is 2 h |df|^2 = 0.1 |df|
    assert abs((losses[0] - losses[1]) / (2 * h) - want) < 0.02 * want + 1e-5 / h


def test_a_training_step_with_muon(gpu):
    from matconvnet_b200 import simplenn, train
    nn, mat, _ = gpu
    import torch
    rng = np.random.default_rng(1)
    net = _net(mat, rng, 333)
    x, c = _data(mat, rng, False, 50, 333)
    net["layers"][-1]["class"] = c
    params = dict(train.default_params(), solver="muon", learning_rate=0.02)
    state = {}
    for step in range(2):
        res = simplenn.vl_simplenn(net, x, 1.0)
        old = [[None if w is None else w.clone() for w in l.get("weights", [])] for l in net["layers"]]
        kept = {k: (dict(v, s1=v["s1"].clone()) if isinstance(v, dict) else v.clone()) for k, v in state.items()}
        state = train.accumulate_gradients(net, res, state, params)
        for i, l in enumerate(net["layers"]):
            for j, w in enumerate(l.get("weights", [])):
                if w is None:
                    continue
                v, der = old[i][j], res[i]["dzdw"][j]
                if j == 0 and l["type"] in ("conv", "fcsoftmaxloss"):
                    nn.solver_update_("muon", v, kept.get((i, j), {}), der, 1.0, params["weight_decay"], 0.02)
                    # alone or with others: the reduction of a product may be cut elsewhere, a few roundings
                    assert float((v - w).norm() / w.norm()) < 1e-6
                else:
                    nn.sgd_update_(v, kept.get((i, j), torch.zeros_like(v)), der, 1.0, params["weight_decay"], params["momentum"], 0.02)
                    assert (v == w).all()
        assert sorted(state) == [(0, 0), (0, 1), (1, 0), (1, 1), (3, 0), (3, 1), (4, 0)]


def test_gradients_into_buckets(gpu):
    from matconvnet_b200 import simplenn
    nn, mat, _ = gpu
    rng = np.random.default_rng(2)
    net = _net(mat, rng, 70, True)
    x, c = _data(mat, rng, True, 12, 70)
    net["layers"][-1]["class"] = c
    specs = simplenn.gradient_specs(net)
    assert [s[0] for s in specs] == ["l4_0", "l4_1", "l1_0", "l1_1", "l0_0", "l0_1"]
    out = {(int(n[1:].split("_")[0]), int(n[-1])): mat.empty(s) for n, s in specs}
    res = simplenn.vl_simplenn(net, x, 1.0, grad_out=out)
    ref = simplenn.vl_simplenn(net, x, 1.0)
    for (i, j), t in out.items():
        assert res[i]["dzdw"][j].data_ptr() == t.data_ptr() and (t.reshape(-1) == ref[i]["dzdw"][j].reshape(-1)).all()
