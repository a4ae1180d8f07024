"""Clusters and distributed shared memory, as an order in the sources that no run can be relied on to show: a CTA may touch
another's shared memory only once all CTAs of the cluster are known to run, and none may leave while another may still reach its own."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pelica_b200", "csrc")
REMOTE = r"map_shared_rank|mapa\.|st\.async|shared::cluster\.[usb]\d|norm_sum<"  # (norm_sum: sums to the other CTAs)


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def kernels(text):
    return {re.search(r"\b(k_\w+)\(", m.group(0)).group(1): m.group(0) for m in re.finditer(r"__global__[^;{]*\{.*?\n}\n", text, re.S)}


def test_every_kernel_of_clusters_is_looked_at():
    found = {n for f in glob.glob(os.path.join(CSRC, "*.cu")) for n, b in kernels(source(os.path.basename(f))).items() if re.search(REMOTE, b)}
    assert found == {"k_rows_sort", "k_block_norm", "k_block_norm_grad"}


def test_a_cluster_has_begun_before_its_first_remote_access():
    body = kernels(source("rows.cu"))["k_rows_sort"]
    first = body.index("map_shared_rank")
    assert "cluster.sync();" in body[:first] and "cluster.sync();" in body[body.rindex("map_shared_rank"):]
    text = source("block_norm.cu")
    helper = {n: re.search(r"void %s\(\) \{(.*?)\n}" % n, text, re.S).group(1) for n in ("norm_cluster_arrive", "norm_cluster_wait")}
    assert "barrier.cluster.arrive" in helper["norm_cluster_arrive"] and "barrier.cluster.wait" in helper["norm_cluster_wait"]
    for name in ("k_block_norm", "k_block_norm_grad"):
        body = kernels(text)[name]
        first = body.index("norm_sum<")
        # every thread arrives once and waits once, outside of the rows' loop and in front of it
        arrive, wait = (body.index("if constexpr (CLUSTER) norm_cluster_%s();" % k) for k in ("arrive", "wait"))
        loop = body.index("for (int t = t0; t < c.T")
        assert arrive < wait < loop < first and not re.search(r"\n  (if [^\n]*)?return", body[:wait]), name
        assert body.count("norm_cluster_") == 2
        assert "cg::this_cluster().sync();" in body[body.rindex("norm_sum<"):], name
