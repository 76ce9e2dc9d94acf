/*
 * A replay on the host of how sample.hip's workgroups take rows by tickets, wait for one another and leave
 * (nanochat_amd/csrc/nc_meeting.h, the code the kernel runs), for any number of launches at once on a device of any size.
 *
 * Every atomic operation is one step of one workgroup, in random order. Launch workgroups start in index order, workgroup i
 * on XCD i % xcds, when that XCD has a place; its places come free one after the other (other work held them) and serve the
 * launches in turn.
 *
 *   replay launches xcds places rows groups meetings patience seed      (patience < 0: waits without bound)
 *
 * prints "ended" when every workgroup has left, every row has one token and all counts are zero again; "stuck" when no
 * workgroup can start and all that run wait without bound; else what is wrong.
 */
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "nc_meeting.h"

using namespace nc;

static const int QUEUES = 8;

struct Word {
    int v = 0;
    int add(int n) { const int was = v; v += n; return was; }
    bool swap(int &expected, int desired) {
        if (v == expected) { v = desired; return true; }
        expected = v;
        return false;
    }
};

struct Launch {
    std::vector<Word> word;
    std::vector<int> tokens;
    int tickets[QUEUES] = {}, done[QUEUES] = {};
    std::vector<int> next;   /* the next workgroup to start on each XCD */
};

enum Step { DRAW, ARRIVE, LOOK, LEAVE, END };

struct Group {
    int launch, index, xcd, row, g, met, reached, seen, patience;
    bool gone;
    Step step;
};

int main(int argc, char **argv) {
    if (argc != 9) return 2;
    const int n = atoi(argv[1]), xcds = atoi(argv[2]), places = atoi(argv[3]), rows = atoi(argv[4]), G = atoi(argv[5]);
    const int meetings = atoi(argv[6]), patience = atoi(argv[7]);
    std::mt19937 rng(atoi(argv[8]));
    const auto below = [&](int k) { return (int)(rng() % (unsigned)k); };
    const int grid = (rows + QUEUES - 1) / QUEUES * QUEUES * G;
    std::vector<Launch> launches(n);
    for (Launch &l : launches) {
        l.word.resize(rows);
        l.tokens.resize(rows, 0);
        for (int x = 0; x < xcds; x++) l.next.push_back(x);
    }
    std::vector<int> held(xcds, places), turn(xcds, 0);   /* places that other work holds; the launch whose turn it is */
    std::vector<int> room(xcds, 0);
    std::vector<Group> live;
    long long left = (long long)n * grid;
    for (long long steps = 0;; steps++) {
        if (left == 0) break;
        if (steps > 400000000LL) { printf("no end\n"); return 0; }
        /* start what has room */
        for (int x = 0; x < xcds; x++) {
            for (int tried = 0; room[x] && tried < n; tried++) {
                const int k = turn[x];
                turn[x] = (k + 1) % n;
                if (launches[k].next[x] >= grid) continue;
                live.push_back(Group{k, launches[k].next[x], x, 0, 0, 0, 0, 0, 0, false, DRAW});
                launches[k].next[x] += xcds;
                room[x]--;
                tried = -1;
            }
        }
        /* another place comes free now and then: at once when nothing else can go on */
        bool waits = patience < 0;
        for (const Group &q : live)
            waits = waits && q.step == LOOK && !(launches[q.launch].word[q.row].v & MT_GIVEN_UP) &&
                    (launches[q.launch].word[q.row].v & MT_ARRIVALS) < q.reached;
        if (live.empty() || waits || below(50) == 0) {
            std::vector<int> some;
            for (int x = 0; x < xcds; x++)
                if (held[x]) some.push_back(x);
            if (!some.empty()) {
                const int x = some[below((int)some.size())];
                held[x]--;
                room[x]++;
                continue;
            }
            if (waits) { printf("stuck\n"); return 0; }
        }
        const int at = below((int)live.size());
        Group &q = live[at];
        Launch &l = launches[q.launch];
        switch (q.step) {
        case DRAW: {
            const int y = q.index % QUEUES, mine = (rows - y + QUEUES - 1) / QUEUES;
            if (q.index / QUEUES >= mine * G) { q.step = END; break; }
            const int ticket = l.tickets[y]++;
            q.row = y + ticket / G * QUEUES;
            q.g = ticket % G;
            if (q.row >= rows) { printf("a ticket past the rows\n"); return 0; }
            q.step = ARRIVE;
            break;
        }
        case ARRIVE:
            q.reached += G;
            q.seen = l.word[q.row].add(1) + 1;
            q.patience = patience < 0 ? 1 : patience;
            q.step = LOOK;
            break;
        case LOOK: {
            if (q.seen < 0) q.seen = l.word[q.row].v;
            const Meeting m = meeting_look(l.word[q.row], q.seen, q.reached, q.patience);
            if (patience < 0) q.patience = 1;
            if (m == MT_WAIT) {
                q.seen = -1;
            } else if (m == MT_GONE) {
                q.gone = true;
                q.step = LEAVE;
            } else if (++q.met == meetings) {
                l.tokens[q.row] += q.g == q.row % G;
                q.step = LEAVE;
            } else {
                q.step = ARRIVE;
            }
            break;
        }
        case LEAVE:
            if (meeting_last(l.word[q.row].add(MT_LEFT), G)) {
                l.tokens[q.row] += q.gone;
                l.word[q.row].v = 0;
                const int y = q.row % QUEUES, mine = (rows - y + QUEUES - 1) / QUEUES;
                if (l.done[y]++ == mine - 1) l.tickets[y] = l.done[y] = 0;
            }
            q.step = END;
            break;
        case END:
            break;
        }
        if (q.step == END) {
            room[q.xcd]++;
            left--;
            live[at] = live.back();
            live.pop_back();
        }
    }
    for (const Launch &l : launches) {
        for (int r = 0; r < rows; r++)
            if (l.tokens[r] != 1 || l.word[r].v) { printf("row %d: %d tokens, word %d\n", r, l.tokens[r], l.word[r].v); return 0; }
        for (int y = 0; y < QUEUES; y++)
            if (l.tickets[y] || l.done[y]) { printf("counts left\n"); return 0; }
    }
    printf("ended\n");
    return 0;
}
