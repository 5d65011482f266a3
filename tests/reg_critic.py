"""td3.RegularisedCritic's definition in 64 bits on the CPU, apart from its code and from the operators' kernels."""
import torch

import reg_oracle as O


def hidden(x, layer, groups, net, rng, weight, bias, gate=None):
    """linear's rows -> dropout -> layer norm per network -> ReLU; gate: where the network under test let the rows through (None: decided here)."""
    if net.training and net.dropout > 0:
        x = torch.where(O.keep(x.shape, net.dropout, rng, layer), x * O.scale_of(net.dropout), 0.0)
    if net.norm:
        v = x.view(x.shape[0], groups, -1)
        v = (v - v.mean(2, keepdim=True)) / torch.sqrt(((v - v.mean(2, keepdim=True)) ** 2).mean(2, keepdim=True) + 1e-5)
        x = v.reshape(x.shape) * weight[:x.shape[1]] + bias[:x.shape[1]]
    return x * (x > 0 if gate is None else gate)


def parameters(net):
    return {k: v.detach().cpu().double().requires_grad_() for k, v in net.named_parameters()}


def forward(net, P, state, action, rng, gates=(None, None)):
    sa = torch.cat([state, action], 1).detach().cpu().double()
    lin = lambda x, n: x @ P[n + ".weight"].t() + P[n + ".bias"]  # noqa: E731
    n = lambda k: (P.get("norm%d.weight" % k), P.get("norm%d.bias" % k))  # noqa: E731
    h = hidden(torch.cat((lin(sa, "fc1"), lin(sa, "fc4")), 1), 0, 2, net, rng, *n(1), gate=gates[0])
    w = h.shape[1] // 2
    h = hidden(torch.cat((lin(h[:, :w], "fc2"), lin(h[:, w:], "fc5")), 1), 1, 2, net, rng, *n(2), gate=gates[1])
    return lin(h[:, :w], "fc3"), lin(h[:, w:], "fc6")


def q1(net, P, state, action, rng, gates=(None, None)):
    sa = torch.cat([state, action], 1)
    sa = sa.cpu().double() if sa.dtype != torch.float64 else sa
    lin = lambda x, n: x @ P[n + ".weight"].t() + P[n + ".bias"]  # noqa: E731
    n = lambda k: (P.get("norm%d.weight" % k), P.get("norm%d.bias" % k))  # noqa: E731
    h = hidden(lin(sa, "fc1"), 0, 1, net, rng, *n(1), gate=gates[0])
    h = hidden(lin(h, "fc2"), 1, 1, net, rng, *n(2), gate=gates[1])
    return lin(h, "fc3")


def check_against_definition(device, dropout, norm, B):
    """Values and gradients of forward and Q1 against the definition.  In 32 bits every product of K terms is off by at most (K + 2) 2^-24 of the sum of its
    terms' sizes, three in a row of at most 256 terms forward, the same backward and B terms over the batch: below 2^-24 (6 * 258 + B) = 1.1e-4 of those sums at B = 300,
    and the sums of sizes are taken to be at most ten times the largest value of the same tensor: 1.1e-3 of it.  A ReLU's gate may fall the other way
    where its input is that close to 0, so the definition is given the gates of the network under test (its value hardly changes there; its gradient would)."""
    from plen_ml_walk_amd import td3 as T
    torch.manual_seed(3 + B)
    net = T.RegularisedCritic(26, 18, dropout, norm, seed=77)
    with torch.no_grad():
        for p in net.parameters():
            if p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    state, action = torch.randn(B, 26), torch.rand(B, 18) * 2 - 1
    t1, t2 = torch.randn(B, 1), torch.randn(B, 1)
    net = net.to(device)
    seen, inner = [], net._hidden
    net._hidden = lambda *a: seen.append(inner(*a)) or seen[-1]
    dev = lambda t: t.to(device)  # noqa: E731
    close = lambda name, got, want: _close(name, got, want)  # noqa: E731

    rng = net.rng.clone().cpu()
    a, b = net(dev(state), dev(action))
    (((a - dev(t1)) ** 2).mean() + ((b - dev(t2)) ** 2).mean()).backward()
    drawn = 1 if dropout > 0 else 0
    assert net.rng.tolist() == [int(rng[0]), int(rng[1]) + drawn]
    P = parameters(net)
    wa, wb = forward(net, P, state, action, rng, [h.detach().cpu() > 0 for h in seen])
    (((wa - t1.double()) ** 2).mean() + ((wb - t2.double()) ** 2).mean()).backward()
    close("q1", a, wa), close("q2", b, wb)
    for k, p in net.named_parameters():
        close(k, p.grad, P[k].grad)

    seen.clear()
    rng = net.rng.clone().cpu()
    act = dev(action).requires_grad_()
    q = net.Q1(dev(state), act)
    (g,) = torch.autograd.grad(q.mean(), act)
    P, want_act = parameters(net), action.double().requires_grad_()
    want = q1(net, P, state.double(), want_act, rng, [h.detach().cpu() > 0 for h in seen])
    (wg,) = torch.autograd.grad(want.mean(), want_act)
    close("Q1", q, want), close("dQ1/da", g, wg)

    # without dropout: no draw, the same values each time
    net.eval()
    with torch.no_grad():
        before = net.rng.tolist()
        a, b = net(dev(state), dev(action))
        assert torch.equal(net(dev(state), dev(action))[0], a) and net.rng.tolist() == before
        wa, wb = forward(net, parameters(net), state, action, rng)
        close("q1 without dropout", a, wa), close("q2 without dropout", b, wb)


def _close(name, got, want):
    got, want = got.detach().cpu().double(), want.detach()
    off, size = float((got - want).abs().max()), float(want.abs().max())
    assert got.shape == want.shape and off <= 1.1e-3 * size + 1e-12, "%s: off by %.3g of %.3g" % (name, off, size)
