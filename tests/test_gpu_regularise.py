"""Learners whose networks have layer norms and dropout (epi_agents_regularise), against a restatement in numpy, and a
network built from the layer operators next to the worlds.

Values are doubles of sizes up to about 10, sums have at most 512 terms (samples) or 256 (units) and nest three deep:
(3 * 512 roundings of 2^-53) * 100 is 2e-11; 1e-10 relative to the larger of 1 and the value is allowed."""
import numpy as np
import pytest

from oracle import layers_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")   # before libepi.so: the two share torch's HIP runtime

TOL = 1e-10


@pytest.fixture(scope="module")
def epi():
    import epidemicsimulator_amd as E
    assert E.lib().epi_device_count() >= 1, "no HIP device: GPU tests must run on the MI355X box"
    return E


def random_state(epi, rng, t):
    pop = int(rng.integers(10_000, 50_000_000))
    i = int(rng.integers(0, max(2, pop // 50))); r = int(rng.integers(0, pop // 10)); d = int(rng.integers(0, pop // 500))
    v = int(rng.integers(0, pop // 20))
    return epi.State(float(pop - i - r - d), float(i), float(r), float(d), float(v), float(rng.integers(50, 100_000)), int(t), 60, 1)


def feed(epi, rng, pools, n, count):
    """The same random transitions into every pool; returned per agent."""
    out = [[] for _ in range(n)]
    for k in range(count):
        trs = [epi.Transition(random_state(epi, rng, k % 60), int(rng.integers(0, 8)), float(rng.normal() * (12.0 if k % 5 == 0 else 2.0)),
                              random_state(epi, rng, k % 60 + 1), bool(rng.random() < 0.15)) for _ in range(n)]
        for p in pools:
            p.observe(trs)
        for a in range(n):
            out[a].append(trs[a])
    return out


class Net:
    """One network in numpy: W1, b1, W2, b2, W3, b3 and the two norms."""

    def __init__(self, weights, norms, eps):
        self.w, self.n, self.eps = [np.array(w) for w in weights], [np.array(v) for v in norms], eps

    def copy(self):
        return Net(self.w, self.n, self.eps)

    def forward(self, x, factors=(None, None)):
        keep = {"x": x}
        h = x
        for l in (0, 1):
            z = h @ self.w[2 * l].T + self.w[2 * l + 1]
            d = z if factors[l] is None else R.apply_factors(z, factors[l])
            y, u, _, r = R.norm_forward(d, self.n[2 * l], self.n[2 * l + 1], self.eps)
            h = np.maximum(y, 0.0)
            keep[l] = (u, r, y, h)
        keep["q"] = h @ self.w[4].T + self.w[5]
        return keep

    def gradients(self, keep, act, err, factors):
        B = len(act)
        dq = np.zeros((B, 8)); dq[np.arange(B), act] = err
        h2, h1 = keep[1][3], keep[0][3]
        gw = [None] * 6; gn = [None] * 4
        gw[4], gw[5] = dq.T @ h2, dq.sum(0)
        dh = err[:, None] * self.w[4][act]
        for l in (1, 0):
            u, r, y, _ = keep[l]
            dy = np.where(y > 0, dh, 0.0)
            dz, gn[2 * l], gn[2 * l + 1] = R.norm_backward(dy, u, r, self.n[2 * l])
            if factors[l] is not None:
                dz = R.apply_factors(dz, factors[l])
            gw[2 * l], gw[2 * l + 1] = dz.T @ (h1 if l else keep["x"]), dz.sum(0)
            if l:
                dh = dz @ self.w[2]
        return [g / B for g in gw], [g / B for g in gn]


def clip(v, c):
    return np.clip(v, -c, c) if np.isfinite(c) else v


class Twin:
    """The learner restated: replay order from a second pool that only samples."""

    def __init__(self, hp, agent, weights, target, norms, tnorms, dropout, eps, seed):
        self.hp, self.agent, self.p, self.seed, self.calls = hp, agent, dropout, seed, 0
        self.on, self.tg = Net(weights, norms, eps), Net(target, tnorms, eps)

    def factors(self, rows):
        if R.threshold(self.p) == 0:
            return None, None
        return tuple(R.factors(rows, self.hp.hidden, self.p, self.seed, (self.agent << 32) + 2 * self.calls + l) for l in (0, 1))

    def errors(self, trs, factors):
        x = np.array([t.s.features() for t in trs]); x2 = np.array([t.s2.features() for t in trs])
        act = np.array([t.a for t in trs]); rew = np.array([t.r for t in trs]); done = np.array([t.done for t in trs])
        keep = self.on.forward(x, factors)
        c = self.hp.clip_q
        best = np.argmax(clip(self.on.forward(x2)["q"], c), axis=1)
        nxt = clip(self.tg.forward(x2)["q"], c)[np.arange(len(trs)), best]
        tgt = clip(np.where(done, rew, rew + self.hp.gamma * nxt), c)
        return keep, act, clip(keep["q"], c)[np.arange(len(trs)), act] - tgt

    def learn(self, trs, steps):
        f = self.factors(len(trs))
        keep, act, err = self.errors(trs, f)
        gw, gn = self.on.gradients(keep, act, err, f)
        self.on.w = [w - self.hp.lr * clip(g, self.hp.grad_clip) for w, g in zip(self.on.w, gw)]
        self.on.n = [w - self.hp.lr * clip(g, self.hp.grad_clip) for w, g in zip(self.on.n, gn)]
        self.calls += 1
        if steps % self.hp.target_update_every == 0:
            self.tg = self.on.copy()
        return float((0.5 * err * err).sum() / len(trs))


def near(what, got, want):
    got, want = np.asarray(got), np.asarray(want)
    off = np.abs(got - want) / np.maximum(1.0, np.abs(want))
    assert np.all(off <= TOL), "%s: %g off" % (what, off.max())


def twins_of(pool, hps, dropout, eps, seed):
    return [Twin(h, a, pool.weights(a), pool.weights(a, True), pool.norms(a), pool.norms(a, True), dropout, eps, seed) for a, h in enumerate(hps)]


def same_networks(pool, twins):
    for a, t in enumerate(twins):
        for target, net in ((False, t.on), (True, t.tg)):
            for g, w in zip(pool.weights(a, target), net.w):
                near("agent %d weights" % a, g, w)
            for g, w in zip(pool.norms(a, target), net.n):
                near("agent %d norms" % a, g, w)


def set_up(epi, hidden, batch, accum, dropout, eps=1e-5, seed=77, n=3, **kw):
    hps = [epi.HyperParams(gamma=0.99 - 0.05 * a, lr=0.05 * (1 + a), clip_q=10.0 - 3.0 * a, grad_clip=1.0 if a != 1 else 0.01, hidden=hidden,
                           batch_size=batch, replay_capacity=4000, target_update_every=2 + a, **kw) for a in range(n)]
    pool, order = epi.Agents(hps, max_grad_accum=accum), epi.Agents(hps, max_grad_accum=accum)
    rng = np.random.default_rng(hidden + batch)
    for a in range(n):   # weights of ordinary size: the reference's start near zero, where every norm is 0 / eps
        W = [rng.normal(size=w.shape) * (0.5 if w.ndim == 2 else 0.1) for w in pool.weights(a)]
        pool.set_weights(a, W)
        pool.set_weights(a, [w + 0.01 for w in W], target=True)
    pool.regularise(dropout, eps, seed)
    for a in range(n):
        pool.set_norms(a, [1 + 0.2 * rng.normal(size=hidden), 0.2 * rng.normal(size=hidden), 1 + 0.2 * rng.normal(size=hidden), 0.2 * rng.normal(size=hidden)])
    return rng, hps, pool, order, twins_of(pool, hps, dropout, eps, seed)


@pytest.mark.parametrize("hidden, batch, accum, dropout", [(16, 4, 2, 0.0), (16, 4, 2, 0.3), (100, 8, 1, 0.1), (128, 128, 4, 0.0), (128, 128, 4, 0.1),
                                                           (130, 6, 2, 0.5), (256, 10, 3, 0.25), (1, 3, 1, 0.0)])
def test_learn_matches_the_restatement(epi, hidden, batch, accum, dropout):
    rng, hps, pool, order, twins = set_up(epi, hidden, batch, accum, dropout)
    trs = feed(epi, rng, (pool, order), 3, batch * accum + 20)
    need, steps = batch * accum, [0, 0, 0]
    for it in range(4):
        steps = [s + int(rng.integers(1, 4)) for s in steps]
        ids = [0, 1, 2] if it != 2 else [2, 0]   # a subset, out of order
        loss, _ = pool.learn([steps[a] for a in ids], [batch] * len(ids), accum, ids)
        for a, got in zip(ids, loss):
            want = twins[a].learn([trs[a][k] for k in order.sample(a, need)], steps[a])
            near("loss", got, want)
        same_networks(pool, twins)
    states = [random_state(epi, rng, 3) for _ in range(3)]
    for target in (False, True):
        q, greedy = pool.q_values(states, target=target)
        for a, s in enumerate(states):
            net = twins[a].tg if target else twins[a].on
            want = clip(net.forward(np.array([s.features()]))["q"][0], hps[a].clip_q)
            near("q", q[a], want)
            assert greedy[a] == int(np.argmax(q[a]))


def test_the_step_follows_the_loss_by_differences(epi):
    """(weights before - after) / lr is the slope of the mean loss with the masks held fixed: central differences of 1e-5
    are off by its square times third derivatives and by 1e-16 / 1e-5 of the loss, together below 1e-6 here."""
    rng, hps, pool, order, twins = set_up(epi, 24, 32, 2, 0.2, n=1)
    hps[0].grad_clip = float("inf")
    pool = epi.Agents(hps, max_grad_accum=2)
    W = [rng.normal(size=w.shape) * (0.5 if w.ndim == 2 else 0.1) for w in pool.weights(0)]
    pool.set_weights(0, W); pool.set_weights(0, W, target=True)
    pool.regularise(0.2, 1e-3, 5)
    twin = twins_of(pool, hps, 0.2, 1e-3, 5)[0]
    trs = feed(epi, rng, (pool, order), 1, 64)[0]
    batch = [trs[k] for k in order.sample(0, 64)]
    f = twin.factors(64)
    keep, act, err = twin.errors(batch, f)
    pool.learn([1], [32], 2)

    def loss():
        q = clip(twin.on.forward(keep["x"], f)["q"], hps[0].clip_q)[np.arange(64), act]
        return float((0.5 * (q - tgt) ** 2).mean())

    tgt = clip(keep["q"], hps[0].clip_q)[np.arange(64), act] - err
    after = pool.weights(0) + pool.norms(0)
    inside = np.abs(keep["q"][np.arange(64), act]) < hps[0].clip_q
    assert inside.all()   # the clamp has no slope of its own here
    for k, w in enumerate(twin.on.w + twin.on.n):
        flat = w.reshape(-1)
        for at in rng.choice(flat.size, size=min(12, flat.size), replace=False):
            was = flat[at]
            flat[at] = was + 1e-5; up = loss()
            flat[at] = was - 1e-5; down = loss()
            flat[at] = was
            slope = (up - down) / 2e-5
            got = (was - after[k].reshape(-1)[at]) / hps[0].lr
            assert abs(got - slope) <= 1e-6 * max(1.0, abs(slope)), (k, at, got, slope)


def test_masks_belong_to_the_agent_not_to_the_call(epi):
    """Two agents learning in one call or in two draw the same masks; another seed draws others."""
    def trained(calls, seed):
        rng, hps, pool, order, _ = set_up(epi, 64, 16, 2, 0.3, n=2)
        pool.regularise(0.3, 1e-5, seed)
        feed(epi, np.random.default_rng(3), (pool,), 2, 40)
        for ids in calls:
            pool.learn([1] * len(ids), [16] * len(ids), 2, ids)
        return [w for a in range(2) for w in pool.weights(a) + pool.norms(a)]

    one = trained([[0, 1], [0, 1]], 9)
    for calls in ([[1], [0], [1], [0]], [[1, 0], [0], [1]]):
        for g, w in zip(trained(calls, 9), one):
            assert np.array_equal(g, w)
    assert any(not np.array_equal(g, w) for g, w in zip(trained([[0, 1], [0, 1]], 10), one))


def test_a_plain_pool_is_what_it_was_beside_a_regularised_one(epi):
    rng = np.random.default_rng(1)
    hps = [epi.HyperParams(hidden=48, batch_size=8, replay_capacity=100) for _ in range(2)]
    pools = [epi.Agents(hps, max_grad_accum=1) for _ in range(3)]
    pools[1].regularise(0.2, 1e-5, 1)
    feed(epi, rng, pools, 2, 30)
    for _ in range(3):
        for p in pools:
            p.learn([1, 1], [8, 8], 1)
    for a in range(2):
        for u, v, w in zip(pools[0].weights(a), pools[2].weights(a), pools[1].weights(a)):
            assert np.array_equal(u, v)
        assert not np.array_equal(pools[0].weights(a)[2], pools[1].weights(a)[2])


def test_refusals(epi):
    pool = epi.Agents([epi.HyperParams(hidden=16, batch_size=4, replay_capacity=50)], max_grad_accum=1)
    for f in (lambda: pool.norms(0), lambda: pool.set_norms(0, [np.ones(16)] * 4), lambda: pool.regularise(1.0), lambda: pool.regularise(-0.1),
              lambda: pool.regularise(float("nan")), lambda: pool.regularise(0.1, 0.0), lambda: pool.regularise(0.1, float("inf"))):
        with pytest.raises(epi.EpiError):
            f()
    pool.regularise(0.1)
    for f in (lambda: pool.set_norms(0, [np.ones(15)] * 4), lambda: pool.set_norms(0, [np.ones(16)] * 3)):
        with pytest.raises(epi.EpiError):
            f()
    g1, b1, g2, b2 = pool.norms(0)
    assert np.all(g1 == 1) and np.all(g2 == 1) and not b1.any() and not b2.any()
    world = epi.WorldToy(epi.HyperParams(), epi.State(0, 0, 0, 0, 0, 10_000.0, 0, 60), batch=2)
    with pytest.raises(epi.EpiError):
        world.regularise(0.1)


def test_regularised_again_starts_afresh(epi):
    """Gains, biases and masks of a second call are those of a first one; the weights stay."""
    hp = epi.HyperParams(hidden=32, batch_size=8, replay_capacity=100, lr=0.05)
    pools = [epi.Agents([hp] * 2, max_grad_accum=1) for _ in range(2)]
    feed(epi, np.random.default_rng(4), pools, 2, 20)
    rng = np.random.default_rng(5)
    W = [rng.normal(size=w.shape) for w in pools[0].weights(0)]
    for p in pools:
        p.regularise(0.2, 1e-5, 9)
        p.learn([1, 1], [8, 8], 1)
    pools[0].learn([2, 2], [8, 8], 1)
    pools[1].learn([2, 2], [8, 8], 1, [1, 0])
    pools[0].regularise(0.3, 1e-4, 6)
    pools[0].regularise(0.2, 1e-5, 9)
    pools[1].regularise(0.2, 1e-5, 9)
    for p in pools:
        for a in range(2):
            for target in (False, True):
                g1, b1, g2, b2 = p.norms(a, target)
                assert np.all(g1 == 1) and np.all(g2 == 1) and not b1.any() and not b2.any()
                p.set_weights(a, W, target)
        p.learn([3, 3], [8, 8], 1)
    for a in range(2):
        for g, w in zip(pools[0].weights(a) + pools[0].norms(a), pools[1].weights(a) + pools[1].norms(a)):
            assert np.array_equal(g, w)
        assert any(not np.array_equal(g, w) for g, w in zip(pools[0].weights(a), W))


def test_a_dropout_that_rounds_to_one_is_refused(epi):
    """The generator takes p in units of 2^-16: 1 - 2^-17 rounds to 1 (halves to even) and would drop every unit of the trained
    pass.  The largest p below it learns."""
    hp = epi.HyperParams(hidden=16, batch_size=4, replay_capacity=50)
    pool = epi.Agents([hp], max_grad_accum=1)
    for p in (1.0 - 2.0 ** -17, 1.0 - 2.0 ** -20, np.nextafter(1.0, 0.0)):
        assert R.threshold(p) == 65536
        with pytest.raises(epi.EpiError):
            pool.regularise(p)
    with pytest.raises(epi.EpiError):
        pool.norms(0)   # a refused call leaves the networks plain
    p = 1.0 - 2.0 ** -16
    assert R.threshold(p) == 65535
    pool.regularise(p, 1e-5, 4)
    feed(epi, np.random.default_rng(2), (pool,), 1, 10)
    loss, _ = pool.learn([1], [4], 1)
    assert np.isfinite(loss[0])
    gains = [1 + 0.1 * np.arange(16.0)] * 4
    pool.set_norms(0, gains)
    for bad in (1.0, 1.0 - 2.0 ** -17):
        with pytest.raises(epi.EpiError):
            pool.regularise(bad)
        assert all(np.array_equal(g, w) for g, w in zip(pool.norms(0), gains))   # and regularised ones as they are


def test_a_world_whose_agents_are_regularised(epi):
    """stepOne until the agents have learned several times, the greedy evaluation on the device, and the same evaluation
    step by step through the agents' Q-values."""
    hp = epi.HyperParams(hidden=64, batch_size=16, learn_every=4, replay_capacity=500, epsilon_decay_steps=50, lr=0.01)
    world = epi.WorldToy(hp, epi.State(0, 0, 0, 0, 0, 10_000.0, 0, 120), countries=epi.ToyConn.C)
    world.regularise(0.1, 1e-5, 3)
    before = [world._pool.norms(a) for a in range(6)]
    for _ in range(90):
        world.step_one(120)
    assert all(any(not np.array_equal(p, q) for p, q in zip(before[a], world._pool.norms(a))) for a in range(6))
    saved = world.snapshot_states()
    world.reset_to_initial()
    out = world.rollout_greedy(25, 120)
    world.restore_states(saved)
    again = epi.WorldToy(hp, epi.State(0, 0, 0, 0, 0, 10_000.0, 0, 120), countries=epi.ToyConn.C)
    again.regularise(0.1, 1e-5, 3)
    for a in range(6):
        again._pool.set_weights(a, world._pool.weights(a))
        again._pool.set_norms(a, world._pool.norms(a))
    # the first world's noise streams stand 90 draws on
    for _ in range(90):
        again.step_actions([[0] * 6], None, 120)
    again.reset_to_initial()
    for k in range(25):
        again.step_one_greedy(120)
        assert [nd.s.i for nd in again.nodes] == list(out["i_series"][k, 0]), "step %d" % k


@pytest.mark.parametrize("hidden, batch", [(64, 130), (128, 9), (100, 33), (256, 2)])
def test_rollouts_of_batched_worlds(epi, hidden, batch):
    """Instances in different states, each asking its node's regularised network on the device, against the same steps with
    the actions that the agents give each instance by itself."""
    import ctypes as C
    from epidemicsimulator_amd import synth
    countries, xy = synth.make_countries(9, 78)
    n, t_max, steps = len(countries), 60, 6
    conn = synth.gravity_dense(countries, xy)
    rng = np.random.default_rng(hidden + batch)
    hp = epi.HyperParams(hidden=hidden)
    pool = epi.Agents([hp] * n)
    pool.regularise(0.2, 1e-4, 1)
    for a in range(n):
        pool.set_weights(a, [rng.normal(size=w.shape) * 0.3 for w in pool.weights(a)])
        pool.set_norms(a, [1 + 0.3 * rng.normal(size=hidden), 0.3 * rng.normal(size=hidden), 1 + 0.3 * rng.normal(size=hidden), 0.3 * rng.normal(size=hidden)])

    def world():
        it = iter([epi.EpidemicEnv(0.25 + 0.01 * k, 0.12, 0.008, 0.04, 5.0, 0.0, c.name, 100 + k, profile=c) for k, c in enumerate(countries)])
        w = epi.WorldToy(hp, epi.State(0, 0, 0, 0, 0, 10_000, 0, t_max, 42), 2, conn, make_env_for=lambda name, pop: next(it), validate=True,
                         countries=countries, batch=batch, learning=False)
        apart = np.random.default_rng(5)
        for _ in range(4):
            st, _ = w.step_arrays(apart.integers(0, 8, (batch, n)), apart.normal(size=(batch, n)), t_max)
        return w, st

    wa, _ = world()
    series, last = np.zeros((steps, batch, n)), np.empty((batch, n), dtype=epi.WorldToy.STATE_DTYPE)
    arr, pk = np.zeros((batch, n), dtype=np.int32), np.zeros((batch, n))
    epi.check(epi.lib().epi_world_rollout_greedy(wa._h, pool._h, C.c_int32(steps), C.c_int32(t_max), series.ctypes.data, arr.ctypes.data,
                                                 pk.ctypes.data, last.ctypes.data))
    wb, st = world()
    asked = set()
    for k in range(steps):
        acts = np.array([pool.q_values([epi.State(*(row[f] for f in ("s", "i", "r", "d", "v", "hosp_cap", "t", "t_max", "seed"))) for row in one])[1]
                         for one in st])
        asked |= set(acts.ravel().tolist())
        st, _ = wb.step_arrays(acts, None, t_max)
        np.testing.assert_array_equal(series[k], st["i"])
    np.testing.assert_array_equal(last, st)
    assert len(asked) > 2   # the networks do choose
    wa.close(); wb.close()


def test_a_network_of_the_operators_beside_batched_worlds(epi):
    """Features of 64 worlds of six countries through linear -> dropout -> norm -> ReLU twice to Q-values with the layer
    operators, a TD loss, its gradients against the formulas in doubles, and the greedy actions back into the worlds."""
    from epidemicsimulator_amd import layers as L
    B, n, h = 64, 6, 128
    world = epi.WorldToy(epi.HyperParams(), epi.State(0, 0, 0, 0, 0, 10_000.0, 0, 60), batch=B)
    rng = np.random.default_rng(8)
    net = Net([rng.normal(size=s) * 0.3 for s in ((h, 7), (h,), (h, h), (h,), (8, h), (8,))], [1 + 0.1 * rng.normal(size=h), 0.1 * rng.normal(size=h)] * 2, 1e-5)
    params = [torch.tensor(v, device="cuda", requires_grad=True) for v in net.w + net.n]
    states, _ = world.step_actions(rng.integers(0, 8, size=(B, n)), None, 60)
    x = np.array([s.features() for row in states for s in row])
    for step in range(3):
        hidden = torch.tensor(x, device="cuda")
        for l in (0, 1):
            z = torch.nn.functional.linear(hidden, params[2 * l], params[2 * l + 1])
            hidden = torch.relu(L.layer_norm(z, params[6 + 2 * l], params[7 + 2 * l], 1e-5, dropout=0.1, seed=4, offset=2 * step + l))
        q = torch.nn.functional.linear(hidden, params[4], params[5])
        act = rng.integers(0, 8, size=B * n)
        tgt = rng.normal(size=B * n)
        chosen = q[torch.arange(B * n, device="cuda"), torch.tensor(act, device="cuda")]
        loss = 0.5 * (chosen - torch.tensor(tgt, device="cuda")).square().mean()
        grads = torch.autograd.grad(loss, params)
        f = tuple(R.factors(B * n, h, 0.1, 4, 2 * step + l) for l in (0, 1))
        keep = net.forward(x, f)
        err = keep["q"][np.arange(B * n), act] - tgt
        gw, gn = net.gradients(keep, act, err, f)
        near("q", q.detach().cpu().numpy(), keep["q"])
        for k, (g, want) in enumerate(zip(grads, gw + gn)):
            near("gradient %d" % k, g.cpu().numpy(), want)
        with torch.no_grad():
            for p, g in zip(params, grads):
                p -= 0.01 * g
        net.w = [p.detach().cpu().numpy() for p in params[:6]]; net.n = [p.detach().cpu().numpy() for p in params[6:]]
        states, _ = world.step_actions(np.argmax(keep["q"], axis=1).reshape(B, n), None, 60)
        x = np.array([s.features() for row in states for s in row])
