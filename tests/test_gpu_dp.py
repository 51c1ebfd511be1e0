"""The product's data-parallel update on the GPU: two ranks (sharing the one GPU of the test
box, gradients exchanged over gloo staged through the host — RCCL needs one GPU per rank)
must reproduce the single-process update when they shard the envs and draw the same global
permutation."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from oracle import tfgraph
from tests import util

pytestmark = pytest.mark.gpu

D, A, T, E, B, NEP = 17, 6, 8, 32, 64, 2
HWC, NACT, NLSTM = (36, 36, 2), 4, 32
# kind -> (nsteps, nenvs over all ranks, global minibatch size); the image cases take a ragged share per rank
# (their global minibatches are not split evenly by the permutation)
SHAPES = {"mlp": (T, E, B), "cnn": (6, 8, 16), "lstm": (6, 8, 2 * 6)}


def _data(kind="mlp"):
    Tk, Ek, _ = SHAPES[kind]
    if kind == "mlp":
        shapes = tfgraph.mlp_param_shapes(D, (64, 64), A, 1, True, "upstream")
        params = util.make_params(shapes, 41, pi_scale=0.5, jitter=0.02)
        ro = util.synthetic_mlp_rollout(np.random.RandomState(42), Tk, Ek, D, A, 1, True, params, nlp_noise=0.2)
        return params, ro
    cell = "lstm" if kind == "lstm" else None
    shapes = tfgraph.cnn_param_shapes(HWC[2], NACT, cell, NLSTM, flat=util.cnn_flat(HWC[0], HWC[1]))
    params = util.make_params(shapes, 51, pi_scale=0.5, jitter=0.002)
    rng = np.random.RandomState(52)
    ro = util.synthetic_cnn_rollout(rng, Tk, Ek, HWC, NACT, params, kind="lstm" if cell else "cnn", nlstm=NLSTM if cell else 0)
    if cell:
        ro["states"] = (0.2 * rng.randn(Ek, 2 * NLSTM)).astype(np.float32)
    return params, ro


def _run_model(kind, params, ro, e0, e1, comm, mode_seed, nbatch_train=None):
    from baselines_amd import hip, spaces
    from baselines_amd.ppo2 import policies
    from baselines_amd.ppo2.common_functions import DeviceRollout, Model
    Tk, _, Bk = SHAPES[kind]
    Bk = nbatch_train or Bk
    dev = lambda a: torch.as_tensor(np.ascontiguousarray(a)).cuda()
    policies.reset_scopes()
    if kind == "mlp":
        model = Model(policy=policies.MlpPolicy64, ob_space=spaces.Box(-1, 1, shape=(D,)), ac_space=spaces.Box(-1, 1, shape=(A,)),
                      nbatch_act=e1 - e0, nbatch_train=Bk, nsteps=Tk, ent_coef=0.0, vf_coef=0.5, max_grad_norm=0.5, comm=comm)
        hyper = (3e-4, 0.2)
    else:
        class SmallLstm(policies.LstmPolicy):
            def __init__(self, *a, **k):
                super().__init__(*a, nlstm=NLSTM, **k)
        model = Model(policy=SmallLstm if kind == "lstm" else policies.CnnPolicy, ob_space=spaces.Box(0, 255, shape=HWC, dtype=np.uint8),
                      ac_space=spaces.Discrete(NACT), nbatch_act=e1 - e0, nbatch_train=Bk, nsteps=Tk, ent_coef=0.01, vf_coef=0.5,
                      max_grad_norm=0.5, upstream_loss=True, comm=comm)
        hyper = (2.5e-4, 0.1)
    model.arena.set_dict(params)
    sl = lambda a: a[:, e0:e1] if a.ndim >= 2 else a[e0:e1]
    d = DeviceRollout(Tk, e1 - e0, dev(sl(ro["obs"])), dev(sl(ro["actions"])), dev(sl(ro["rewards"])), dev(sl(ro["values"])),
                      dev(sl(ro["neglogpacs"])), dev(sl(ro["dones"])), dev(ro["last_values"][e0:e1]), dev(ro["last_dones"][e0:e1]),
                      states=dev(ro["states"][e0:e1]) if kind == "lstm" else None)
    d.advs_gae, d.returns, d.advs_ori = hip.gae(d.rewards, d.values, d.dones, d.last_values, d.last_dones, 0.99, 0.95)
    d.advs = d.advs_ori.reshape(Tk, e1 - e0)
    np.random.seed(mode_seed)
    losses = model.train_on_rollout(hyper[0], hyper[1], d, NEP, Bk).cpu().numpy()
    model.check_faults()
    theta = model.arena.theta.cpu().numpy()
    model.close()
    return losses, theta


def _worker(rank, world, port, kind, out):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    from baselines_amd.common.mpi_adam import DataParallel
    comm = DataParallel("global")
    params, ro = _data(kind)
    e0, e1 = comm.env_range(SHAPES[kind][1])
    losses, theta = _run_model(kind, params, ro, e0, e1, comm, 5)
    assert comm.check_synced(torch.from_numpy(theta).cuda())
    if rank == 0:
        out.put((losses, theta))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("kind", ["mlp", "cnn", "lstm"])
def test_two_ranks_reproduce_single_process_update(kind):
    """"global" mode: both ranks draw the single process's minibatch order over all envs and work on their shares (the
    ownership filter and the shares' statistics run on the device; the shares of the image cases are ragged); the
    parameters after two epochs must be the single process's up to summation order.  cnn + LSTM: env-sequence
    minibatches with one global env order (baselines/ppo2/ppo2.py:124-136)."""
    assert torch.cuda.is_available()
    params, ro = _data(kind)
    l1, t1 = _run_model(kind, params, ro, 0, SHAPES[kind][1], None, 5)
    l2, t2 = util.run_ranks(_worker, 2, args=(kind,))
    np.testing.assert_allclose(l2, l1, rtol=5e-5, atol=2e-7)
    t0 = util.flatten_params(params, type("S", (), {"nparams": t1.size, "vars": _vars(kind)})())
    moved = np.abs(t1 - t0).max()
    assert np.abs(t1 - t2).max() <= (2e-6 if kind == "mlp" else 5e-6), np.abs(t1 - t2).max()
    assert moved > 1e-4


def _vars(kind="mlp"):
    from baselines_amd import _lib, hip
    if kind == "mlp":
        return hip.PolicySpec(_lib.POLICY_MLP, _lib.DIST_GAUSSIAN, A, 1, ob_dim=D, hidden=(64, 64), order=_lib.ORDER_UPSTREAM).vars
    if kind == "cnn":
        return hip.PolicySpec(_lib.POLICY_CNN, _lib.DIST_CATEGORICAL, NACT, 1, ob_hwc=HWC).vars
    return hip.PolicySpec(_lib.POLICY_CNN_LSTM, _lib.DIST_CATEGORICAL, NACT, 1, ob_hwc=HWC, nlstm=NLSTM).vars


# ---- the kernels of the global-permutation mode ---------------------------------------------------------
@pytest.mark.parametrize("Ng,Bg,lo,hi,stride", [(4096, 1024, 1024, 2048, 1024), (6000, 1500, 0, 6000, 1500), (8 * 2048 + 40, 4106, 3000, 3001, 64),
                                                (40000, 10000, 39000, 40000, 10000), (40000, 10000, 5000, 25000, 4000)])
def test_ownership_filter_and_share_statistics(Ng, Bg, lo, hi, stride):
    """ppo2hip_filter_owned_i32 / ppo2hip_adv_stats_owned against NumPy on a random global order: per minibatch the owned
    entries in list order, re-based; their count; {sum a, sum a^2, n} of the share.  The last case hands over list
    slots too small for the shares: the fault word says so and the lists are cut, not overrun."""
    from baselines_amd import hip
    rng = np.random.RandomState(Ng + lo)
    order = rng.permutation(Ng).astype(np.int32)
    nmb = Ng // Bg
    Tl = 8 if (hi - lo) % 8 == 0 else 1
    El = (hi - lo) // Tl
    advs = rng.randn(Tl, El)
    d_advs = torch.as_tensor(advs).cuda()
    d_idx = torch.as_tensor(order).cuda()
    out = torch.full((nmb * stride + 7,), -7, dtype=torch.int32, device="cuda")
    counts = torch.zeros(nmb, dtype=torch.int32, device="cuda")
    hip.filter_owned(d_idx, Bg, nmb, lo, hi, out, stride, counts)
    stats = hip.adv_stats_owned(d_advs, d_idx, Bg, nmb, lo, hi, Tl, El).cpu().numpy()
    bits = hip.take_faults(raise_on_fault=False)
    got, cnt = out.cpu().numpy(), counts.cpu().numpy()
    assert np.all(got[nmb * stride:] == -7)
    overflow = False
    for j in range(nmb):
        mb = order[j * Bg:(j + 1) * Bg]
        want = mb[(mb >= lo) & (mb < hi)] - lo
        assert cnt[j] == want.size
        keep = min(want.size, stride)
        overflow |= want.size > stride
        np.testing.assert_array_equal(got[j * stride:j * stride + keep], want[:keep])
        a = advs.T.ravel()[want]          # env-major flat sample s sits at [s % T, s // T]
        np.testing.assert_allclose(stats[j], [a.sum(), (a * a).sum(), want.size], rtol=1e-12, atol=1e-12)
        pad = got[j * stride + keep:min((j + 1) * stride, j * stride + want.size + 64)]
        assert np.all(pad == 0) or want.size >= stride
    assert bool(bits) == overflow


def test_epoch_over_shares_with_one_owner_equals_epoch_dp():
    """ppo2hip_ppo_epoch_shares on a one-rank RCCL communicator that owns every sample (shares = whole minibatches)
    against ppo2hip_ppo_epoch_dp on the same list: bit for bit."""
    from baselines_amd import hip
    from baselines_amd.ppo2 import policies
    params, ro = _data("mlp")
    results = []
    for shares in (False, True):
        from baselines_amd import spaces
        from baselines_amd.ppo2.common_functions import DeviceRollout, Model
        dev = lambda a: torch.as_tensor(np.ascontiguousarray(a)).cuda()
        policies.reset_scopes()
        model = Model(policy=policies.MlpPolicy64, ob_space=spaces.Box(-1, 1, shape=(D,)), ac_space=spaces.Box(-1, 1, shape=(A,)),
                      nbatch_act=E, nbatch_train=B, nsteps=T, ent_coef=0.0, vf_coef=0.5, max_grad_norm=0.5)
        model.arena.set_dict(params)
        d = DeviceRollout(T, E, dev(ro["obs"]), dev(ro["actions"]), dev(ro["rewards"]), dev(ro["values"]), dev(ro["neglogpacs"]),
                          dev(ro["dones"]), dev(ro["last_values"]), dev(ro["last_dones"]))
        _, d.returns, d.advs_ori = hip.gae(d.rewards, d.values, d.dones, d.last_values, d.last_dones, 0.99, 0.95, want_advs=False)
        d.advs = d.advs_ori.reshape(T, E)
        rref = hip.RolloutRef(model.spec, d.obs, d.actions, d.returns, d.values, d.neglogpacs, d.advs, T, E)
        idx = dev(np.random.RandomState(3).permutation(T * E).astype(np.int32))
        nmb = T * E // B
        losses = torch.zeros((nmb, 8), device="cuda")
        comm = hip.NativeComm(hip.NativeComm.unique_id(), 0, 1)
        if shares:
            stats = hip.adv_stats_owned(d.advs, idx, B, nmb, 0, T * E, T, E)
            local, counts = torch.empty(T * E, dtype=torch.int32, device="cuda"), torch.empty(nmb, dtype=torch.int32, device="cuda")
            hip.filter_owned(idx, B, nmb, 0, T * E, local, B, counts)
            assert counts.cpu().tolist() == [B] * nmb and torch.equal(local, idx)
            hip.ppo_epoch_shares(model.spec, model.loss_desc, model.arena.theta, model.grads, model.adam_m, model.adam_v, rref, local,
                                 B, [B] * nmb, stats, 0.2, 1.0 / B, 3e-4, 1, losses, model._workspace(B), model._adam_scratch,
                                 max_grad_norm=0.5, comm=comm)
        else:
            stats = hip.adv_stats(d.advs, idx, B, nmb, T, E)
            hip.ppo_epoch(model.spec, model.loss_desc, model.arena.theta, model.grads, model.adam_m, model.adam_v, rref, idx, B,
                          stats, 0.2, 3e-4, 1, losses, model._workspace(B), model._adam_scratch, max_grad_norm=0.5, comm=comm,
                          grad_scale=1.0)
        torch.cuda.synchronize()
        results.append((model.arena.theta.clone(), losses.clone(), model.adam_v.clone(), stats.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)


# ---- running statistics exchanged over the data-parallel group -----------------------------------------
def _rms_data(rank):
    rng = np.random.RandomState(0)
    p = [rng.randn(3, 2), rng.randn(4, 2), rng.randn(5, 2)]
    q = [rng.randn(6, 2) * 3 + 1, rng.randn(7, 2) * 3 + 1, rng.randn(8, 2) * 3 + 1]
    return (p, q)[rank], p + q


def _rms_worker(rank, world, port, out):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    from baselines_amd.common.mpi_adam import DataParallel
    from baselines_amd.common.mpi_running_mean_std import RunningMeanStd
    rms = RunningMeanStd(epsilon=0.0, shape=(2,), comm=DataParallel("mpi"))
    mine, _ = _rms_data(rank)
    for x in mine:
        rms.update(x)
    if rank == 0:
        out.put((rms.mean, rms.std, rms.state.cpu().numpy()))
    dist.barrier()
    dist.destroy_process_group()


def test_mpi_running_mean_std_two_ranks():
    """The reference's own distributed check (baselines/common/mpi_running_mean_std.py:85-107): two ranks fed
    different data end with the statistics of the concatenated data."""
    from oracle import envwrap
    mean, std, state = util.run_ranks(_rms_worker, 2)
    _, everything = _rms_data(0)
    allx = np.concatenate(everything)
    # the reference compares with allclose against mean / std of the whole; std floors its variance at 1e-2
    assert np.allclose(mean, allx.mean(0)) and np.allclose(std, np.sqrt(np.maximum(allx.var(0), 1e-2)), atol=1e-6)
    o = envwrap.MpiRunningMeanStd(epsilon=0.0, shape=(2,))
    o.update(allx)
    np.testing.assert_allclose(state, np.concatenate([o._sum, o._sumsq, [o._count]]), rtol=1e-13)


def test_mpi_running_mean_std_single_process():
    """:46-63 of the same file: three updates equal one pass; totals against the oracle to float64 rounding,
    mean / std (float32 in the reference's graph) exactly where the totals agree."""
    from baselines_amd.common.mpi_running_mean_std import RunningMeanStd
    from oracle import envwrap
    rng = np.random.RandomState(1)
    for shape in ((), (2,), (5, 3)):
        xs = [(rng.randn(*((n,) + shape)) * 2 + 0.5).astype(np.float32 if n != 4 else np.float64) for n in (3, 4, 500)]
        rms, o = RunningMeanStd(shape=shape), envwrap.MpiRunningMeanStd(shape=shape)
        for x in xs:
            rms.update(x)
            o.update(x)
        st = rms.state.cpu().numpy()
        np.testing.assert_allclose(st, np.concatenate([o._sum.ravel(), o._sumsq.ravel(), [o._count]]), rtol=1e-13)
        np.testing.assert_allclose(rms.mean, o.mean, rtol=1e-6, atol=1e-7)
        np.testing.assert_allclose(rms.std, o.std, rtol=1e-6)
        assert rms.mean.dtype == np.float32 and rms.mean.shape == shape


# ---- AdamW over ranks -----------------------------------------------------------------------------------
ADAMW_SHAPES = ((33, 17), (17,), (3000,), (), (5, 0))


def _adamw_run(comm, grads, dtype, bits, clip):
    """Five steps of MpiAdamW from rank-dependent parameters that rank 0's replace."""
    from baselines_amd.common.mpi_adam import MpiAdamW
    rng = np.random.RandomState(7 + (comm.rank if comm else 0))
    params = [torch.tensor(np.asarray(rng.randn(*s), np.float32)).cuda().to(dtype) for s in ADAMW_SHAPES]
    opt = MpiAdamW(params, comm=comm, state_bits=bits, max_grad_norm=clip, decay=[1, 0, 1, 0, 1], grad_dtype=torch.float32)
    opt.sync()
    for g in grads:
        opt.update([torch.tensor(x).cuda() for x in g], 1e-2)
    opt.check_synced()
    return [p.float().cpu().numpy() for p in params] + [opt.plan.norm[:1].cpu().numpy()]


def _adamw_grads(rank):
    """Multiples of 1/64: sums over two ranks and halves of them are exact."""
    rng = np.random.RandomState(90 + rank)
    return [[np.asarray(rng.randint(-200, 200, s) / 64.0, np.float32) for s in ADAMW_SHAPES] for _ in range(5)]


def _adamw_worker(rank, world, port, dtype, bits, clip, out):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    from baselines_amd.common.mpi_adam import DataParallel
    got = _adamw_run(DataParallel("mpi"), _adamw_grads(rank), getattr(torch, dtype), bits, clip)
    if rank == 0:
        out.put(got)
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("dtype,bits,clip", [("float32", 32, 0.0), ("bfloat16", 8, 0.5)])
def test_mpi_adamw_over_two_ranks(dtype, bits, clip):
    """The mean of two ranks' gradients, clipped by its norm: bit for bit the steps that a single process takes with it."""
    mean = [[np.asarray((a + b) / 2, np.float32) for a, b in zip(x, y)] for x, y in zip(_adamw_grads(0), _adamw_grads(1))]
    want = _adamw_run(None, mean, getattr(torch, dtype), bits, clip)
    got = util.run_ranks(_adamw_worker, 2, args=(dtype, bits, clip))
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
