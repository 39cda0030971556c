"""The categorical depth loss of the training step on the labels that the training step makes: pixels without a LiDAR return take no part."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_pixels_without_a_return_have_no_gradient(mmt_lib):
    """depth_labels() writes bin 0 for a pixel without a return (or out of range), a valid depth begins at bin 1: loss and gradient of
    the step's own logits, with clouds of a few points, against cross entropy in 64 bits over the labelled pixels alone."""
    from mm_training_amd.dp import TrainStep, make_config, synthetic_batch
    from mm_training_amd.ops.train_targets import depth_labels
    torch.manual_seed(0)
    dev = torch.device("cuda", 0)
    cfg = dict(make_config("tiny"), depth_loss="nll")
    ts = TrainStep(cfg, dev)
    batch = list(synthetic_batch(cfg, dev, seed=1))
    for few in (None, 40, 0):
        clouds = batch[2] if few is None else [c[:max(few, 1)].clone() for c in batch[2]]
        if few == 0:
            for c in clouds:
                c[:, :3] = 1e4                                 # no return anywhere
        seen, plain = [], ts.model.forward

        def forward(*args, **kwargs):
            out = plain(*args, **kwargs)
            out[1].retain_grad()
            seen.append(out[1])
            return out

        ts.model.forward = forward
        try:
            np.random.seed(5)
            flips = np.random.uniform(size=batch[0].shape[0] * batch[0].shape[1] * batch[0].shape[2]) > 0.5
            np.random.seed(5)
            _, _, depth_loss = ts.forward_loss([batch[0], batch[1], clouds] + batch[3:])
        finally:
            ts.model.forward = plain
        depth_loss.backward()
        logits, = seen
        H, W = batch[0].shape[-2:]
        mats = batch[1]
        onehot, bins = depth_labels(clouds, mats["extrinsics"][:, 0], mats["intrin_mats"][:, 0], mats["bda_mat"], (H, W), ts.downsample, ts.dbound,
                                    ts.depth_channels, return_bins=True, flipped=torch.from_numpy(flips).to(torch.uint8).cuda() if ts.augment else None)
        bins = bins.cpu().long()
        given = bins > 0
        assert few == 0 or bool(given.any())
        assert not bool(given.all()) and bool((onehot.max(1).values > 0).all())
        x = logits.detach().cpu().double().permute(0, 2, 3, 1).reshape(-1, ts.depth_channels).requires_grad_(True)
        count = max(int(given.sum()), 1)
        want = -3.0 * x.log_softmax(1).gather(1, bins[:, None])[:, 0][given].sum() / count
        want.backward()
        assert abs(float(depth_loss.detach()) - float(want.detach())) <= 1e-5 * max(1.0, abs(float(want.detach())))
        got = torch.zeros_like(x) if logits.grad is None else logits.grad.cpu().double().permute(0, 2, 3, 1).reshape(-1, ts.depth_channels)
        assert not got[~given].any(), "a pixel without a label is trained"
        assert ((got - x.grad).abs() <= 1e-4 * x.grad.abs() + 1e-8).all()
