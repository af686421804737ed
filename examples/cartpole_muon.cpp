// The training loop of cartpole.cpp with the block matrices on Muon, and back on Adam
// for its last iterations.
#include <cstdio>

#include "mg/envs/cartpole.h"
#include "mg/ppo.h"

int main() {
    const uint32_t N = 4096;  // environments
    const uint32_t T = 32;    // steps per rollout

    Gym<CartPole> gym(N);
    PPOModel<CartPole> model(gym, 128, 4, 2, 3e-4f, T);
    model.useMuon(3e-3f);  // the matrices' own learning rate; the rest stays on Adam at 3e-4

    for (int it = 0; it < 20; it++) {
        if (it == 15) model.useAdam();
        model.collect();
        model.train();
        if (it % 5 == 4) {
            LossStats s = model.lastStats();
            std::printf("iter %3d  entropy %.3f  kl %.4f\n", it, s.entropy, s.approxKl);
        }
    }
    return 0;
}
